// rope.cu - rotary positions of query and key heads (include/sapphire_attention.h).
//
//   (a, b) -> (a cos - b sin, a sin + b cos),  angle = position * f_i
//
// The reference tabulates cos and sin per position on the host
// (src/transformer/rope.c:19-37).  Here a frequency is kept as a 64-bit
// fixed-point fraction of a turn, F_i = round(f_i / 2pi * 2^64): position *
// F_i mod 2^64 is the phase, reduced exactly by the overflow of an integer
// product, good to 2^-32 of a turn at any 32-bit position, and sincospi takes
// the reduced half turns.  No table is read, so a call moves its heads once in
// and once out.
#include <cmath>
#include <cstring>

#include "attention.cuh"

struct sapphire_rope {
    kernel_context_t *ctx = nullptr;
    sapphire_rope_config_t cfg{};
    unsigned long long *freq = nullptr;   // device, [rot_dim / 2]
    float amplitude = 1.0f;
};

namespace {

constexpr int kRopeMaxDim = 512;
constexpr int kThreads = 256;
constexpr int kUnit = 8;                  // values of a head that a thread takes from each half
constexpr int kMaxTokens = 16;            // tokens of one block (its cos and sin rows in shared memory)

struct RopeHeads {
    const void *in;
    void *out;
    long long in_ts, in_hs, out_ts, out_hs;
};

struct RopeParams {
    const unsigned long long *freq;
    const int *positions;
    RopeHeads q, k;
    int tokens, q_heads, heads;           // heads: query and key heads together
    int head_dim, half;                   // half: rot_dim / 2
    int block_tokens, block_heads;
    int units;                            // threads of one head: pair units, then copy units
    int pair_units;
    float amplitude, direction;           // direction: 1, or -1 to turn back
    bool wide, copy_tail;
};

// A block turns block_tokens tokens x block_heads heads; a thread owns one
// unit of a head (8 values of the first half and their 8 partners, or 8
// interleaved values) and walks down the heads.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeParams p) {
    extern __shared__ float2 turn[];      // [block_tokens][half] (cos, sin)
    const int t0 = blockIdx.x * p.block_tokens, nt = min(p.block_tokens, p.tokens - t0);
    const int tid = threadIdx.y * blockDim.x + threadIdx.x, nthreads = blockDim.x * blockDim.y;
    for (int i = tid; i < nt * p.half; i += nthreads) {
        const int t = i / p.half, m = i - t * p.half;
        const unsigned long long phase = (unsigned long long)(long long)p.positions[t0 + t] * p.freq[m];
        float s, c;
        sincospif((float)(int)(phase >> 32) * 0x1p-31f, &s, &c);
        turn[i] = make_float2(c * p.amplitude, s * p.amplitude * p.direction);
    }
    __syncthreads();
    const int h0 = blockIdx.y * p.block_heads, nh = min(p.block_heads, p.heads - h0);
    const int u = threadIdx.x;
    for (int r = threadIdx.y; r < nt * nh; r += blockDim.y) {
        const int t = r / nh;
        int h = h0 + r - t * nh;
        const RopeHeads &x = h < p.q_heads ? p.q : p.k;
        if (h >= p.q_heads) h -= p.q_heads;
        const T *in = static_cast<const T *>(x.in) + (long long)(t0 + t) * x.in_ts + (long long)h * x.in_hs;
        T *out = static_cast<T *>(x.out) + (long long)(t0 + t) * x.out_ts + (long long)h * x.out_hs;
        if (u >= p.pair_units) {          // behind the rotated part
            const int d0 = 2 * p.half + (u - p.pair_units) * kUnit;
            if (d0 + kUnit <= p.head_dim) {
                float a[kUnit];
                load_row<T, kUnit>(in + d0, p.wide, a);
                store_row<T, kUnit>(out + d0, p.wide, a);
            } else {
                for (int d = d0; d < p.head_dim; ++d) out[d] = in[d];
            }
        } else if (kInterleaved) {
            const int m0 = u * (kUnit / 2), n = min(kUnit / 2, p.half - m0);
            const float2 *cs = turn + t * p.half + m0;
            if (n == kUnit / 2) {
                float a[kUnit], y[kUnit];
                load_row<T, kUnit>(in + 2 * m0, p.wide, a);
#pragma unroll
                for (int j = 0; j < kUnit / 2; ++j) {
                    y[2 * j] = a[2 * j] * cs[j].x - a[2 * j + 1] * cs[j].y;
                    y[2 * j + 1] = a[2 * j] * cs[j].y + a[2 * j + 1] * cs[j].x;
                }
                store_row<T, kUnit>(out + 2 * m0, p.wide, y);
            } else {
                for (int j = 0; j < n; ++j) {
                    const float a = to_f32(in[2 * (m0 + j)]), b = to_f32(in[2 * (m0 + j) + 1]);
                    out[2 * (m0 + j)] = from_f32<T>(a * cs[j].x - b * cs[j].y);
                    out[2 * (m0 + j) + 1] = from_f32<T>(a * cs[j].y + b * cs[j].x);
                }
            }
        } else {
            const int m0 = u * kUnit, n = min(kUnit, p.half - m0);
            const float2 *cs = turn + t * p.half + m0;
            if (n == kUnit) {
                float a[kUnit], b[kUnit];
                load_row<T, kUnit>(in + m0, p.wide, a);
                load_row<T, kUnit>(in + p.half + m0, p.wide, b);
#pragma unroll
                for (int j = 0; j < kUnit; ++j) {
                    const float x0 = a[j], x1 = b[j];
                    a[j] = x0 * cs[j].x - x1 * cs[j].y;
                    b[j] = x0 * cs[j].y + x1 * cs[j].x;
                }
                store_row<T, kUnit>(out + m0, p.wide, a);
                store_row<T, kUnit>(out + p.half + m0, p.wide, b);
            } else {
                for (int j = 0; j < n; ++j) {
                    const float a = to_f32(in[m0 + j]), b = to_f32(in[p.half + m0 + j]);
                    out[m0 + j] = from_f32<T>(a * cs[j].x - b * cs[j].y);
                    out[p.half + m0 + j] = from_f32<T>(a * cs[j].y + b * cs[j].x);
                }
            }
        }
    }
}

// Frequencies in radians a position (include/sapphire_attention.h).
double rope_frequency(const sapphire_rope_config_t &c, int i) {
    const double pi = 3.14159265358979323846;
    const double f = pow(c.theta, -2.0 * i / c.rot_dim);
    if (c.scaling == SAPPHIRE_ROPE_LINEAR) return f / c.factor;
    if (c.scaling == SAPPHIRE_ROPE_BANDED) {
        const double r = c.original_context * f / (2 * pi);
        const double s = fmin(fmax((r - c.turns_slow) / (c.turns_fast - c.turns_slow), 0.0), 1.0);
        return (1 - s) * (f / c.factor) + s * f;
    }
    if (c.scaling == SAPPHIRE_ROPE_YARN) {
        auto pair = [&](double turns) {
            return c.rot_dim * log(c.original_context / (2 * pi * turns)) / (2 * log(c.theta));
        };
        const double lo = fmax(floor(pair(c.turns_fast)), 0.0);
        const double hi = fmin(ceil(pair(c.turns_slow)), c.rot_dim - 1.0);
        const double g = fmin(fmax((i - lo) / fmax(hi - lo, 1e-3), 0.0), 1.0);
        return (1 - g) * f + g * (f / c.factor);
    }
    return f;
}

// Radians a position as a fraction of a turn in units of 2^-64.
unsigned long long turn_fraction(double f) {
    const long double turns = (long double)f / (2 * 3.14159265358979323846264338327950288L);
    const long double frac = turns - floorl(turns);
    const long double x = frac * 18446744073709551616.0L;
    return x >= 18446744073709551615.0L ? 0ull : (unsigned long long)(x + 0.5L);
}

const char *rope_config_error(const sapphire_rope_config_t &c) {
    if (c.head_dim <= 0 || c.head_dim > kRopeMaxDim || c.head_dim % 2) return "head_dim must be even, 2 to 512";
    if (c.rot_dim <= 0 || c.rot_dim > c.head_dim || c.rot_dim % 2) return "rot_dim must be even and at most head_dim";
    if (c.layout != SAPPHIRE_ROPE_HALF && c.layout != SAPPHIRE_ROPE_INTERLEAVED) return "unknown layout";
    if (c.scaling < SAPPHIRE_ROPE_UNSCALED || c.scaling > SAPPHIRE_ROPE_YARN) return "unknown scaling";
    if (!(c.theta > 1.0) || !std::isfinite(c.theta)) return "theta must be above 1";
    if (c.scaling != SAPPHIRE_ROPE_UNSCALED && (!(c.factor >= 1.0) || !std::isfinite(c.factor)))
        return "factor must be at least 1";
    if (c.scaling == SAPPHIRE_ROPE_BANDED || c.scaling == SAPPHIRE_ROPE_YARN) {
        if (c.original_context <= 0) return "original_context must be positive";
        if (!(c.turns_slow > 0) || !(c.turns_fast > c.turns_slow) || !std::isfinite(c.turns_fast))
            return "turns_slow and turns_fast must be positive and in this order";
    }
    if (!(c.attention_factor > 0) || !std::isfinite(c.attention_factor)) return "attention_factor must be positive";
    return nullptr;
}

template <typename T>
cudaError_t launch_rope(const RopeParams &p, bool interleaved, dim3 grid, dim3 block, size_t smem, cudaStream_t st) {
    if (interleaved)
        rope_kernel<T, true><<<grid, block, smem, st>>>(p);
    else
        rope_kernel<T, false><<<grid, block, smem, st>>>(p);
    return cudaGetLastError();
}

}  // namespace

extern "C" SAPPHIRE_API sapphire_rope_t *sapphire_rope_create(kernel_context_t *ctx,
                                                              const sapphire_rope_config_t *cfg) {
    if (!ctx || !cfg) {
        LOG_ERROR("sapphire_rope_create: NULL argument");
        return nullptr;
    }
    sapphire_rope_config_t c = *cfg;
    if (c.rot_dim == 0) c.rot_dim = c.head_dim;
    if (c.turns_slow == 0) c.turns_slow = 1.0;
    if (c.turns_fast == 0) c.turns_fast = c.scaling == SAPPHIRE_ROPE_YARN ? 32.0 : 4.0;
    if (c.attention_factor == 0)
        c.attention_factor = c.scaling == SAPPHIRE_ROPE_YARN && c.factor > 0 ? 0.1 * log(c.factor) + 1.0 : 1.0;
    if (const char *why = rope_config_error(c)) {
        ctx_fail(ctx, "sapphire_rope_create", "%s", why);
        return nullptr;
    }
    std::lock_guard<std::recursive_mutex> lk(ctx->exec_mutex);
    if (!ctx->initialized) {
        ctx_fail(ctx, "sapphire_rope_create", "context not initialized");
        return nullptr;
    }
    AttnDevice g(ctx->device);
    unsigned long long f[kRopeMaxDim / 2];
    for (int i = 0; i < c.rot_dim / 2; ++i) f[i] = turn_fraction(rope_frequency(c, i));
    sapphire_rope_t *r = new (std::nothrow) sapphire_rope();
    if (!r) return nullptr;
    r->ctx = ctx;
    r->cfg = c;
    r->amplitude = (float)c.attention_factor;
    const size_t bytes = (size_t)c.rot_dim / 2 * sizeof f[0];
    cudaError_t e = cudaMalloc((void **)&r->freq, bytes);
    if (e == cudaSuccess) e = cudaMemcpy(r->freq, f, bytes, cudaMemcpyHostToDevice);
    if (e != cudaSuccess) {
        ctx_fail(ctx, "sapphire_rope_create", "frequency upload failed: %s", cudaGetErrorString(e));
        cudaGetLastError();
        if (r->freq) cudaFree(r->freq);
        delete r;
        return nullptr;
    }
    return r;
}

extern "C" SAPPHIRE_API void sapphire_rope_destroy(sapphire_rope_t *rope) {
    if (!rope) return;
    {
        std::lock_guard<std::recursive_mutex> lk(rope->ctx->exec_mutex);
        AttnDevice g(rope->ctx->device);
        cudaFree(rope->freq);             // waits for the work that uses it
    }
    delete rope;
}

extern "C" SAPPHIRE_API int sapphire_rope_device(sapphire_rope_t *rope, const sapphire_rope_args_t *a) {
    const char *who = "sapphire_rope_device";
    if (!rope || !a) {
        LOG_ERROR("%s: NULL argument", who);
        return -1;
    }
    kernel_context_t *ctx = rope->ctx;
    const sapphire_rope_config_t &c = rope->cfg;
    std::lock_guard<std::recursive_mutex> lk(ctx->exec_mutex);
    const size_t size = io_size(a->dtype);
    if (!size) {
        ctx_fail(ctx, who, "q and k must be F32, BF16 or F16");
        return -1;
    }
    if (a->tokens < 0 || a->q_heads < 0 || a->k_heads < 0 || a->q_heads > 65536 || a->k_heads > 65536) {
        ctx_fail(ctx, who, "tokens and heads must not be negative, nor heads above 65536");
        return -1;
    }
    if (a->tokens == 0 || a->q_heads + a->k_heads == 0) return 0;
    RopeParams p{};
    p.tokens = a->tokens;
    p.q_heads = a->q_heads;
    p.heads = a->q_heads + a->k_heads;
    p.head_dim = c.head_dim;
    p.half = c.rot_dim / 2;
    p.freq = rope->freq;
    p.positions = a->positions;
    p.amplitude = rope->amplitude;
    p.direction = a->inverse ? -1.0f : 1.0f;
    auto heads = [&](const void *in, void *out, int n, long long its, long long ihs, long long ots, long long ohs) {
        RopeHeads h;
        h.in = in;
        h.out = out;
        h.in_hs = ihs ? ihs : c.head_dim;
        h.out_hs = ohs ? ohs : c.head_dim;
        h.in_ts = its ? its : (long long)n * c.head_dim;
        h.out_ts = ots ? ots : (long long)n * c.head_dim;
        return h;
    };
    p.q = heads(a->q, a->q_out, a->q_heads, a->q_token_stride, a->q_head_stride, a->q_out_token_stride,
                a->q_out_head_stride);
    p.k = heads(a->k, a->k_out, a->k_heads, a->k_token_stride, a->k_head_stride, a->k_out_token_stride,
                a->k_out_head_stride);
    if (!on_device(ctx, who, "positions", a->positions)) return -1;
    p.wide = true;
    p.copy_tail = false;
    const RopeHeads *sides[2] = {a->q_heads ? &p.q : nullptr, a->k_heads ? &p.k : nullptr};
    for (const RopeHeads *h : sides) {
        if (!h) continue;
        if (!on_device(ctx, who, h == &p.q ? "q" : "k", h->in)) return -1;
        if (h->out != h->in && !on_device(ctx, who, h == &p.q ? "q_out" : "k_out", h->out)) return -1;
        if (h->out == h->in && (h->in_ts != h->out_ts || h->in_hs != h->out_hs)) {
            ctx_fail(ctx, who, "a rotation in place needs equal strides");
            return -1;
        }
        p.copy_tail = p.copy_tail || h->out != h->in;
        p.wide = p.wide && rows_aligned(h->in, h->in_ts, h->in_hs, size) && rows_aligned(h->out, h->out_ts, h->out_hs, size);
    }
    const bool inter = c.layout == SAPPHIRE_ROPE_INTERLEAVED;
    // The partner half and the tail start on 16 bytes too.
    p.wide = p.wide && (c.rot_dim * (int)size) % 16 == 0 && (inter || (p.half * (int)size) % 16 == 0);
    p.pair_units = inter ? (p.half + kUnit / 2 - 1) / (kUnit / 2) : (p.half + kUnit - 1) / kUnit;
    const int tail = p.copy_tail ? (c.head_dim - c.rot_dim + kUnit - 1) / kUnit : 0;
    p.units = p.pair_units + tail;
    const int rows = std::max(1, kThreads / p.units);
    // A block takes as many tokens as give each of its rows about four heads;
    // few tokens are cut by heads instead, each block computing its own turns.
    AttnDevice g(ctx->device);
    const int sms = sm_count(ctx->device);
    p.block_heads = p.heads;
    p.block_tokens = std::min(kMaxTokens, std::max(1, 4 * rows / p.heads));
    while (p.block_tokens > 1 && (p.tokens + p.block_tokens - 1) / p.block_tokens < 2 * sms) p.block_tokens /= 2;
    if (p.block_tokens == 1)
        while (p.block_heads > rows && (long long)p.tokens * ((p.heads + p.block_heads - 1) / p.block_heads) < 2 * sms)
            p.block_heads = (p.block_heads + 1) / 2;
    const dim3 grid((p.tokens + p.block_tokens - 1) / p.block_tokens, (p.heads + p.block_heads - 1) / p.block_heads);
    const dim3 block(p.units, rows);
    const size_t smem = (size_t)p.block_tokens * p.half * sizeof(float2);
    cudaError_t e = a->dtype == DTYPE_F32    ? launch_rope<float>(p, inter, grid, block, smem, ctx->stream)
                    : a->dtype == DTYPE_BF16 ? launch_rope<__nv_bfloat16>(p, inter, grid, block, smem, ctx->stream)
                                             : launch_rope<__half>(p, inter, grid, block, smem, ctx->stream);
    if (e != cudaSuccess) {
        ctx_fail(ctx, who, "launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
