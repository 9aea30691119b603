// rope.cu - rotary positions of query and key heads (include/sapphire_attention.h).
//
//   (a, b) -> (a cos - b sin, a sin + b cos),  angle = position * f_i
//
// The reference tabulates cos and sin per position on the host
// (src/transformer/rope.c:19-37).  Here a frequency is kept as a 64-bit
// fixed-point fraction of a turn, F_i = round(f_i / 2pi * 2^64): position *
// F_i mod 2^64 is the phase, reduced exactly by the overflow of an integer
// product and good to 2^-32 of a turn at any 32-bit position; as the fp32 half
// turns that sincospi takes it is good to 2^-26 of one.  No table is read, so a call moves its heads once in
// and once out, and is bound by that: 16381 tokens x 40 bf16 heads of 128 take
// 59 us, 5.7 TB/s.  Single tokens cost a launch.
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
// Values of a head that a thread takes (from each half where these are paired):
// 8, or 4 where the halves have a multiple of 4 and not of 8, whose ends would
// go value by value (4991 tokens x 20 bf16 heads, 40 of 80 turned: 44 -> 12 us).
constexpr int rope_unit(bool interleaved, int half) { return !interleaved && half % 8 == 4 ? 4 : 8; }
// Tokens of a thread in flight, and the next ones behind them: 64 bytes of 16-bit values any way.
constexpr int rope_batch(bool interleaved, int unit) { return interleaved || unit == 4 ? 4 : 2; }
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
    int row_heads;                        // heads that the rows of a block take at a time
    int pair_units;
    float amplitude, direction;           // direction: 1, or -1 to turn back
    bool wide, copy_tail;
};

// A block turns block_tokens tokens x its heads.  A thread owns one unit of a
// head (kUnit values of the first half and their partners, 8 interleaved values,
// or kUnit values behind the rotated part) and one row of blockDim.y: head h0 + y %
// row_heads, token y / row_heads; it walks down the tokens and then the heads.
// The block's cos and sin lie in shared memory as [token][pair of pairs][unit],
// so that neighbouring units read neighbouring 16 bytes.
template <typename T, bool kInterleaved, int kUnit>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeParams p) {
    constexpr int kPairs = kInterleaved ? kUnit / 2 : kUnit, kBatch = rope_batch(kInterleaved, kUnit);
    extern __shared__ float4 turn[];
    pdl_trigger();
    pdl_wait();
    const int t0 = blockIdx.x * p.block_tokens, nt = min(p.block_tokens, p.tokens - t0), units = p.pair_units;
    const int tid = threadIdx.y * blockDim.x + threadIdx.x, nthreads = blockDim.x * blockDim.y;
    const int u = threadIdx.x, token_rows = blockDim.y / p.row_heads;
    const int h0 = blockIdx.y * p.block_heads, h_end = min(h0 + p.block_heads, p.heads);
    const int ty = threadIdx.y / p.row_heads, hy = threadIdx.y - ty * p.row_heads;
    const bool tail = u >= units;         // behind the rotated part
    const int m0 = u * kPairs, d_tail = 2 * p.half + (u - units) * kUnit;
    const int at_a = tail ? d_tail : kInterleaved ? 2 * m0 : m0, at_b = p.half + m0;
    const bool short_unit = tail ? d_tail + kUnit > p.head_dim : m0 + kPairs > p.half;
    auto input = [&](int h, int t) {
        const RopeHeads &x = h >= p.q_heads ? p.k : p.q;
        return static_cast<const T *>(x.in) + (long long)(t0 + t) * x.in_ts + (long long)(h >= p.q_heads ? h - p.q_heads : h) * x.in_hs;
    };
    auto output = [&](int h, int t) {
        const RopeHeads &x = h >= p.q_heads ? p.k : p.q;
        return static_cast<T *>(x.out) + (long long)(t0 + t) * x.out_ts + (long long)(h >= p.q_heads ? h - p.q_heads : h) * x.out_hs;
    };
    // kBatch tokens of a head at a time, the next ones' loads in flight.
    struct Batch {
        Raw<T, kUnit> a[kBatch], b[kInterleaved ? 1 : kBatch];
    };
    auto load = [&](Batch &x, int h, int t1) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int t = t1 + k * token_rows;
            if (t >= nt) continue;
            const T *in = input(h, t);
            x.a[k].load(in + at_a, p.wide);
            if constexpr (!kInterleaved)
                if (!tail) x.b[k].load(in + at_b, p.wide);
        }
    };
    int h = h0 + hy, t1 = ty;
    bool more = !short_unit && h < h_end && t1 < nt;
    Batch x;
    if (more) load(x, h, t1);
    for (int i = tid; i < nt * p.half; i += nthreads) {
        const int t = i / p.half, m = i - t * p.half, j = m % kPairs;
        const unsigned long long phase = (unsigned long long)(long long)p.positions[t0 + t] * p.freq[m];
        float s, c;
        sincospif((float)(int)(phase >> 32) * 0x1p-31f, &s, &c);
        reinterpret_cast<float2 *>(turn)[((t * (kPairs / 2) + j / 2) * units + m / kPairs) * 2 + j % 2] =
            make_float2(c * p.amplitude, s * p.amplitude * p.direction);
    }
    __syncthreads();
    if (short_unit) {
        // The end of a part: value by value.
        for (; h < h_end; h += p.row_heads)
            for (int t = ty; t < nt; t += token_rows) {
                const T *a = input(h, t);
                T *o = output(h, t);
                if (tail) {
                    for (int d = d_tail; d < p.head_dim; ++d) o[d] = a[d];
                    continue;
                }
                for (int m = m0; m < p.half; ++m) {
                    const float2 cs = reinterpret_cast<const float2 *>(turn)[((t * (kPairs / 2) + (m - m0) / 2) * units + u) * 2 + (m - m0) % 2];
                    const int i = kInterleaved ? 2 * m : m, j = kInterleaved ? 2 * m + 1 : p.half + m;
                    const float v0 = to_f32(a[i]), v1 = to_f32(a[j]);
                    o[i] = from_f32<T>(v0 * cs.x - v1 * cs.y);
                    o[j] = from_f32<T>(v0 * cs.y + v1 * cs.x);
                }
            }
        return;
    }
    while (more) {
        int h2 = h, t2 = t1 + kBatch * token_rows;
        if (t2 >= nt) {
            t2 = ty;
            h2 += p.row_heads;
        }
        more = h2 < h_end;
        Batch next;
        if (more) load(next, h2, t2);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int t = t1 + k * token_rows;
            if (t >= nt) continue;
            T *out = output(h, t);
            if (!tail) {
                float a[kUnit], b[kUnit];
                x.a[k].get(a);
                if constexpr (!kInterleaved) x.b[k].get(b);
#pragma unroll
                for (int j = 0; j < kPairs; j += 2) {
                    const float4 cs = turn[(t * (kPairs / 2) + j / 2) * units + u];
                    const float c2[4] = {cs.x, cs.y, cs.z, cs.w};
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float &v = kInterleaved ? a[(2 * (j + i)) & (kUnit - 1)] : a[j + i], &w = kInterleaved ? a[(2 * (j + i) + 1) & (kUnit - 1)] : b[j + i];
                        const float v0 = v, v1 = w;
                        v = v0 * c2[2 * i] - v1 * c2[2 * i + 1];
                        w = v0 * c2[2 * i + 1] + v1 * c2[2 * i];
                    }
                }
                x.a[k].set(a);
                if constexpr (!kInterleaved) {
                    x.b[k].set(b);
                    x.b[k].store(out + at_b, p.wide);
                }
            }
            x.a[k].store(out + at_a, p.wide);
        }
        x = next;
        h = h2;
        t1 = t2;
    }
}

// Frequencies in radians a position (include/sapphire_attention.h), in the
// host's 64-bit significands: a double's 2^-53 of one would be 2^-25 of a turn at
// position 2^31.
constexpr long double kPi = 3.14159265358979323846264338327950288L;
long double rope_frequency(const sapphire_rope_config_t &c, int i) {
    const long double f = powl(c.theta, -2.0L * i / c.rot_dim);
    if (c.scaling == SAPPHIRE_ROPE_LINEAR) return f / c.factor;
    if (c.scaling == SAPPHIRE_ROPE_BANDED) {
        const long double r = c.original_context * f / (2 * kPi);
        const long double s = fminl(fmaxl((r - c.turns_slow) / ((long double)c.turns_fast - c.turns_slow), 0.0L), 1.0L);
        return (1 - s) * (f / c.factor) + s * f;
    }
    if (c.scaling == SAPPHIRE_ROPE_YARN) {
        auto pair = [&](long double turns) {
            return c.rot_dim * logl(c.original_context / (2 * kPi * turns)) / (2 * logl(c.theta));
        };
        const long double lo = fmaxl(floorl(pair(c.turns_fast)), 0.0L);
        const long double hi = fminl(ceill(pair(c.turns_slow)), c.rot_dim - 1.0L);
        const long double g = fminl(fmaxl((i - lo) / fmaxl(hi - lo, 1e-3L), 0.0L), 1.0L);
        return (1 - g) * f + g * (f / c.factor);
    }
    return f;
}

// Radians a position as a fraction of a turn in units of 2^-64.
unsigned long long turn_fraction(long double f) {
    const long double turns = f / (2 * kPi);
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
cudaError_t launch_rope(const RopeParams &p, bool interleaved, int unit, dim3 grid, dim3 block, size_t smem, cudaStream_t st) {
    if (interleaved) return launch_pdl(rope_kernel<T, true, 8>, grid, block, smem, st, p);
    if (unit == 4) return launch_pdl(rope_kernel<T, false, 4>, grid, block, smem, st, p);
    return launch_pdl(rope_kernel<T, false, 8>, grid, block, smem, st, p);
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
    const bool inter = c.layout == SAPPHIRE_ROPE_INTERLEAVED;
    const int unit = rope_unit(inter, p.half), align = std::min(16, unit * (int)size);
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
        p.wide = p.wide && rows_aligned(h->in, h->in_ts, h->in_hs, size, align) &&
                 rows_aligned(h->out, h->out_ts, h->out_hs, size, align);
    }
    // The partner half and the tail start there too.
    p.wide = p.wide && (c.rot_dim * (int)size) % align == 0 && (inter || (p.half * (int)size) % align == 0);
    p.pair_units = inter ? (p.half + unit / 2 - 1) / (unit / 2) : (p.half + unit - 1) / unit;
    const int tail = p.copy_tail ? (c.head_dim - c.rot_dim + unit - 1) / unit : 0;
    const int units = p.pair_units + tail;      // threads of one head
    const int rows = std::max(1, kThreads / units);
    // A block's rows are heads of one token, evenly divided where there are
    // more than rows, or heads of several tokens; each row then walks down
    // tokens (four batches of them) and heads, so a block's cos and sin serve
    // every head.  Where that gives an SM fewer than eight blocks, a row takes
    // fewer tokens, then a block fewer heads, computing its own turns (1507
    // tokens x 96 heads of 256: 47 us with whole blocks, 31 us so).
    AttnDevice g(ctx->device);
    const int batch = rope_batch(inter, unit);
    auto cut = [](int n, int most) { return (n + (n + most - 1) / most - 1) / ((n + most - 1) / most); };
    p.block_heads = p.heads;
    p.row_heads = cut(p.heads, rows);
    const int token_rows = rows / p.row_heads;
    p.block_tokens = std::min(kMaxTokens, 4 * batch * token_rows);
    const long long wanted = 8ll * sm_count(ctx->device);
    auto blocks = [&] {
        return (long long)((p.tokens + p.block_tokens - 1) / p.block_tokens) * ((p.heads + p.block_heads - 1) / p.block_heads);
    };
    while (blocks() < wanted) {
        if (p.block_tokens > batch * token_rows) p.block_tokens = (p.block_tokens + 1) / 2;
        else if (p.block_heads > p.row_heads) p.block_heads = cut(p.block_heads, (p.block_heads + 1) / 2);
        else if (p.block_tokens > 1) p.block_tokens = (p.block_tokens + 1) / 2;
        else break;
    }
    p.row_heads = cut(p.block_heads, p.row_heads);
    const dim3 grid((p.tokens + p.block_tokens - 1) / p.block_tokens, (p.heads + p.block_heads - 1) / p.block_heads);
    const dim3 block(units, p.row_heads * std::min(token_rows, p.block_tokens));
    const size_t smem = (size_t)p.block_tokens * p.pair_units * (inter ? unit / 2 : unit) * sizeof(float2);
    cudaError_t e = a->dtype == DTYPE_F32    ? launch_rope<float>(p, inter, unit, grid, block, smem, ctx->stream)
                    : a->dtype == DTYPE_BF16 ? launch_rope<__nv_bfloat16>(p, inter, unit, grid, block, smem, ctx->stream)
                                             : launch_rope<__half>(p, inter, unit, grid, block, smem, ctx->stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        ctx_fail(ctx, who, "launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
