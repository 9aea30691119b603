// kv_cache.cu - the paged key-value cache (include/sapphire_attention.h):
// keys and values stored as they are or quantised, and read back dense.
//
// The block formulas are those of kernel_quantize_q8_0 / _q4_0 (quant.cu),
// every float step one IEEE-rounded operation, so a row's codes and scales are
// the same numbers; only their order inside a row differs (8 x nb words of
// four codes, include/sapphire_attention.h).
//
// Both directions move each value once in and once out and are bound by that:
// 8192 fp16 tokens of 8 KV heads of 128 into Q8_0 pages and 65193 back out take
// 94 us, 5.0 TB/s, in two launches.  A step of one token a sequence costs its
// launch.
#include <cstring>

#include "attention.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kUnit = 8;          // consecutive values of a row that one thread takes: words 2t and 2t + 1 of a block
constexpr int kMaxTokens = 32;    // tokens of one block

struct KvParams {
    KvLayout l;
    KvRows r;
    int block_tokens, units;      // units: threads of one row
    int row_heads;                // of K and V together, that the rows of a block take at a time
    bool wide;
    int *err;
};

// Where a token lives, in units of 16 bytes from a head's first row (row) and
// from its first page (page), and its slot; slot -1: nowhere.
struct KvPlace {
    unsigned row, page;
    int slot;
};

// The place of row `i` of ragged sequences.  A row outside the table or on a
// page outside the cache sets the error word.
__device__ __forceinline__ KvPlace kv_place(const KvLayout &l, const KvRows &r, int i, int *err) {
    const KvPlace nowhere = {0, 0, -1};
    int s, j;
    if (r.cu_tokens) {
        // The sequence whose rows hold i: the largest s with cu_tokens[s] <= i.
        int lo = 0, hi = r.sequences;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (__ldg(r.cu_tokens + mid) <= i) lo = mid;
            else hi = mid - 1;
        }
        if (lo == r.sequences) return nowhere;               // behind the last sequence
        s = lo;
        j = i - __ldg(r.cu_tokens + s);
        if (j < 0) return nowhere;                           // before the first
    } else {
        s = i;
        j = 0;
    }
    const long long pos = (long long)j + (r.start ? __ldg(r.start + s) : 0);
    const long long page = pos < 0 ? -1 : pos / l.page_size;
    if (page < 0 || page >= r.table_stride) {
        atomicOr(err, kErrCache);
        return nowhere;
    }
    const int id = __ldg(r.page_table + (long long)s * r.table_stride + page);
    if (id < 0 || id >= l.num_pages) {
        atomicOr(err, kErrCache);
        return nowhere;
    }
    KvPlace at;
    at.slot = (int)(pos - page * l.page_size);
    at.page = (unsigned)id * (unsigned)(l.page_bytes >> 4);
    at.row = at.page + (unsigned)(at.slot * (l.row_bytes >> 4));
    return at;
}

// Lanes of one 32-value block: four neighbours, `mask` their bits.
__device__ __forceinline__ float block_max(float v, unsigned mask) {
    v = fmaxf(v, __shfl_xor_sync(mask, v, 1));
    return fmaxf(v, __shfl_xor_sync(mask, v, 2));
}

// The bits of a block's largest magnitude, at least kInfBits where a value is
// infinite or none: magnitudes are ordered like their bits.
template <typename T>
struct Magnitude {
    static constexpr uint32_t kInfBits = sizeof(T) == 4 ? 0x7f800000u : 0x7c00u;
};
template <>
struct Magnitude<__nv_bfloat16> {
    static constexpr uint32_t kInfBits = 0x7f80u;
};
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t m;
    asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    return m;
}
template <typename T>
__device__ __forceinline__ uint32_t block_magnitude(const Raw8<T> &x, unsigned mask) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(x.v);
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) m = max(m, w[j] & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) m = max(m, __shfl_xor_sync(mask, m, o));
        return m;
    } else {
#pragma unroll
        for (int j = 0; j < kUnit / 2; ++j) m = max_u16x2(m, w[j] & 0x7fff7fffu);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) m = max_u16x2(m, __shfl_xor_sync(mask, m, o));
        return max(m & 0xffffu, m >> 16);
    }
}
// Four values' signs as bytes of ones or zeros.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t permute_signs(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "n"(kSel));        // a selector's top bit spreads the sign
    return r;
}
template <typename T>
__device__ __forceinline__ uint32_t sign_bytes(const Raw8<T> &x, int k) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(x.v);
    if constexpr (sizeof(T) == 4)
        return __byte_perm(permute_signs<0x00fb>(w[4 * k], w[4 * k + 1]), permute_signs<0x00fb>(w[4 * k + 2], w[4 * k + 3]), 0x5410);
    else
        return permute_signs<0xfdb9>(w[2 * k], w[2 * k + 1]);
}

// Codes of 8 values as the two words' bytes (Q8_0: one uint32 each; Q4_0: 16
// bits each); returns the block's scale.
template <typename T>
__device__ __forceinline__ float quantize_q8(const Raw8<T> &raw, unsigned mask, uint32_t (&w)[2]) {
    float x[kUnit];
    raw.get(x);
    const uint32_t bits = block_magnitude(raw, mask);
    if (bits < Magnitude<T>::kInfBits) {
        const T top = *reinterpret_cast<const T *>(&bits);        // (its low half for 16-bit types)
        const float d = __fdiv_rn(to_f32(top), 127.0f);
        const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
        if (id < INFINITY) {
            // |x| id is at most 127 and a rounding, so no code is clamped.  Half
            // away from zero is the whole part of |t| + 1/2: both sums truncate,
            // so neither rounds a value below a half up.
            uint32_t n[kUnit];
#pragma unroll
            for (int j = 0; j < kUnit; ++j)
                n[j] = __float_as_uint(__fadd_rz(__fadd_rz(fabsf(__fmul_rn(x[j], id)), 0.5f), 8388608.0f));
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                // 128 + n or 128 - n in each byte: neither carries.
                const uint32_t m = __byte_perm(__byte_perm(n[4 * k], n[4 * k + 1], 0x0040), __byte_perm(n[4 * k + 2], n[4 * k + 3], 0x0040), 0x5410);
                const uint32_t minus = sign_bytes(raw, k);
                w[k] = ((0x80808080u + m) & ~minus) | ((0x80808080u - m) & minus);
            }
            return d;
        }
    }
    // A block with an infinity or a NaN (not the largest, code 0), or with a
    // scale whose reciprocal is infinite.
    float a = 0.0f;
#pragma unroll
    for (int j = 0; j < kUnit; ++j) a = fmaxf(a, fabsf(x[j]));
    const float d = __fdiv_rn(block_max(a, mask), 127.0f);
    const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        w[k] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float t = roundf(__fmul_rn(x[4 * k + j], id));
            w[k] |= (uint32_t)(((t != t) ? 0 : (t > 127.0f ? 127 : (t < -127.0f ? -127 : (int)t))) + 128) << (8 * j);
        }
    }
    return d;
}
__device__ __forceinline__ float quantize_q4(const float (&x)[kUnit], unsigned mask, uint32_t (&w)[2]) {
    // The value of largest magnitude, the first of the block on ties.  A NaN
    // never compares above, so it is not chosen.
    float a = 0.0f, m = 0.0f;
#pragma unroll
    for (int j = 0; j < kUnit; ++j)
        if (fabsf(x[j]) > a) {
            a = fabsf(x[j]);
            m = x[j];
        }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const float b = __shfl_xor_sync(mask, a, o), n = __shfl_xor_sync(mask, m, o);
        const bool lower = (threadIdx.x & o) != 0;           // the other lane's values come first
        if (b > a || (b == a && lower)) {
            a = b;
            m = n;
        }
    }
    const float d = __fdiv_rn(m, -8.0f);
    const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        w[k] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // a NaN becomes 0; the truncating sum leaves the whole part
            const float t = fminf(fmaxf(__fadd_rn(__fmul_rn(x[4 * k + j], id), 8.5f), 0.0f), 15.0f);
            w[k] |= (__float_as_uint(__fadd_rz(t, 8388608.0f)) & 15u) << (4 * j);
        }
    }
    return d;
}

// Rows of a block: K and V of every KV head of block_tokens tokens.  A thread
// owns one unit of a row and one row of blockDim.y: K or V of KV head y %
// row_heads (V behind K), token y / row_heads; it walks down the tokens, kBatch
// at a time with their loads in flight together, and then the heads.  The four
// threads of a quantised block are neighbours in a warp (units is a multiple of 4).
constexpr int kBatch = 2;

// The type of a dense cache's values (unused for quantised ones).
template <int kCache>
struct KvType {
    using type = float;
};
template <>
struct KvType<DTYPE_BF16> {
    using type = __nv_bfloat16;
};
template <>
struct KvType<DTYPE_F16> {
    using type = __half;
};

// What a thread needs of its head: its unit of the block's first token, and the
// head's rows and scales in the first page.
template <typename T>
struct KvHead {
    T *io;
    long long ts;
    uint8_t *rows, *scales;
};
template <typename T>
__device__ __forceinline__ KvHead<T> kv_head(const KvParams &p, int c, int t0, int d0) {
    const bool is_v = c >= p.l.kv_heads;
    const int h = is_v ? c - p.l.kv_heads : c;
    KvHead<T> r;
    r.ts = is_v ? p.r.v_ts : p.r.k_ts;
    r.io = static_cast<T *>(is_v ? p.r.v : p.r.k) + (long long)t0 * r.ts + (long long)h * (is_v ? p.r.v_hs : p.r.k_hs) + d0;
    uint8_t *chunk = p.l.pages + (unsigned long long)h * p.l.chunk_bytes;
    r.rows = chunk + (is_v ? p.l.v_off : 0);
    r.scales = chunk + (is_v ? p.l.vs_off : p.l.ks_off);
    return r;
}
__device__ __forceinline__ uint8_t *kv_at(uint8_t *p, unsigned off16) { return p + (unsigned long long)off16 * 16; }

template <typename T, int kCache>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvParams p) {
    __shared__ KvPlace place[kMaxTokens];
    pdl_trigger();
    pdl_wait();
    const int t0 = blockIdx.x * p.block_tokens, nt = min(p.block_tokens, p.r.tokens - t0);
    const int tid = threadIdx.y * blockDim.x + threadIdx.x;
    const int u = threadIdx.x, token_rows = blockDim.y / p.row_heads, heads = 2 * p.l.kv_heads;
    const int ty = threadIdx.y / p.row_heads, cy = threadIdx.y - ty * p.row_heads;
    const int nb = p.l.head_dim / 32, b = u >> 2, word = 2 * (u & 3);
    const unsigned mask = 0xfu << (tid & 28);
    bool looked = false;
    for (int c = cy; c < heads; c += p.row_heads) {
        const KvHead<T> r = kv_head<T>(p, c, t0, u * kUnit);
        // kBatch tokens at a time, the next ones' loads in flight.
        Raw8<T> x[kBatch];
        const T *io = r.io + ty * r.ts;
        const long long step = token_rows * r.ts;
        auto load = [&](int t) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k, io += step)
                if (t + k * token_rows < nt) x[k].load(io, p.wide);
        };
        load(ty);
        if (!looked) {                    // the first rows do not wait for their places
            if (tid < nt) place[tid] = kv_place(p.l, p.r, t0 + tid, p.err);
            __syncthreads();
            looked = true;
        }
        for (int t = ty; t < nt; t += kBatch * token_rows) {
            Raw8<T> y[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) y[k] = x[k];
            load(t + kBatch * token_rows);
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (t + k * token_rows >= nt) continue;
                const KvPlace at = place[t + k * token_rows];
                if (at.slot < 0) continue;
                uint8_t *row = kv_at(r.rows, at.row);
                if constexpr (kCache == DTYPE_Q8_0 || kCache == DTYPE_Q4_0) {
                    uint32_t q[2];
                    float d;
                    if (kCache == DTYPE_Q8_0) {
                        d = quantize_q8(y[k], mask, q);
                        reinterpret_cast<uint32_t *>(row)[word * nb + b] = q[0];
                        reinterpret_cast<uint32_t *>(row)[(word + 1) * nb + b] = q[1];
                    } else {
                        float v[kUnit];
                        y[k].get(v);
                        d = quantize_q4(v, mask, q);
                        reinterpret_cast<uint16_t *>(row)[word * nb + b] = (uint16_t)q[0];
                        reinterpret_cast<uint16_t *>(row)[(word + 1) * nb + b] = (uint16_t)q[1];
                    }
                    if ((u & 3) == 0) reinterpret_cast<float *>(kv_at(r.scales, at.page))[at.slot * p.l.scale_stride + b] = d;
                } else {
                    using C = typename KvType<kCache>::type;
                    float v[kUnit];
                    y[k].get(v);
                    Raw8<C> z;
                    z.set(v);
                    z.store(reinterpret_cast<C *>(row) + u * kUnit, true);
                }
            }
        }
    }
}

template <typename T, int kCache>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvParams p) {
    constexpr bool kQuant = kCache == DTYPE_Q8_0 || kCache == DTYPE_Q4_0;
    using C = typename KvType<kCache>::type;
    __shared__ KvPlace place[kMaxTokens];
    pdl_trigger();
    pdl_wait();
    const int t0 = blockIdx.x * p.block_tokens, nt = min(p.block_tokens, p.r.tokens - t0);
    const int tid = threadIdx.y * blockDim.x + threadIdx.x;
    const int u = threadIdx.x, token_rows = blockDim.y / p.row_heads, heads = 2 * p.l.kv_heads;
    const int ty = threadIdx.y / p.row_heads, cy = threadIdx.y - ty * p.row_heads;
    const int nb = p.l.head_dim / 32, b = u >> 2, word = 2 * (u & 3);
    const int at_u = kCache == DTYPE_Q8_0 ? 4 * (word * nb + b) : kCache == DTYPE_Q4_0 ? 2 * (word * nb + b) : u * kUnit * (int)sizeof(C);
    // What a thread loads of a row: a block's scale and the bytes of two words, or values.
    struct Unit {
        bool ok;
        float d;
        uint32_t w[2];
        Raw8<C> x;
    };
    if (tid < nt) place[tid] = kv_place(p.l, p.r, t0 + tid, p.err);
    __syncthreads();
    for (int c = cy; c < heads; c += p.row_heads) {
        const KvHead<T> r = kv_head<T>(p, c, t0, u * kUnit);
        uint8_t *const rows = r.rows + at_u, *const scales = r.scales + 4 * b;
        Unit x[kBatch];
        auto load = [&](int t) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                x[k].ok = false;
                if (t + k * token_rows >= nt) continue;
                const KvPlace at = place[t + k * token_rows];
                x[k].ok = at.slot >= 0;
                if (!x[k].ok) continue;
                const uint8_t *row = kv_at(rows, at.row);
                if constexpr (kQuant) {
                    x[k].d = *reinterpret_cast<const float *>(kv_at(scales, at.page) + at.slot * p.l.scale_stride * 4);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        x[k].w[j] = kCache == DTYPE_Q8_0 ? reinterpret_cast<const uint32_t *>(row)[j * nb] : reinterpret_cast<const uint16_t *>(row)[j * nb];
                } else {
                    x[k].x.load(reinterpret_cast<const C *>(row), true);
                }
            }
        };
        load(ty);
        T *io = r.io + ty * r.ts;
        const long long step = token_rows * r.ts;
        for (int t = ty; t < nt; t += kBatch * token_rows) {
            Unit y[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) y[k] = x[k];
            load(t + kBatch * token_rows);
#pragma unroll
            for (int k = 0; k < kBatch; ++k, io += step) {
                if (!y[k].ok) continue;
                float v[kUnit];
                if constexpr (kQuant) {
                    // 2^23 + code by its bytes, and the offset off again: exact
#pragma unroll
                    for (int j = 0; j < kUnit; ++j) {
                        const uint32_t q = kCache == DTYPE_Q8_0 ? __byte_perm(y[k].w[j / 4], 0x4b000000u, 0x7440 + (j & 3))
                                                                : ((y[k].w[j / 4] >> (4 * (j & 3))) & 15u) | 0x4b000000u;
                        v[j] = __fmul_rn(__fadd_rn(__uint_as_float(q), kCache == DTYPE_Q8_0 ? -8388736.0f : -8388616.0f), y[k].d);
                    }
                } else {
                    y[k].x.get(v);
                }
                Raw8<T> z;
                z.set(v);
                z.store(io, p.wide);
            }
        }
    }
}

template <typename T, int kCache>
cudaError_t launch_kv(const KvParams &p, bool write, dim3 grid, dim3 block, cudaStream_t st) {
    return write ? launch_pdl(kv_write_kernel<T, kCache>, grid, block, 0, st, p)
                 : launch_pdl(kv_read_kernel<T, kCache>, grid, block, 0, st, p);
}
template <typename T>
cudaError_t launch_kv(tensor_dtype_t cache, const KvParams &p, bool write, dim3 grid, dim3 block, cudaStream_t st) {
    switch (cache) {
        case DTYPE_F32: return launch_kv<T, DTYPE_F32>(p, write, grid, block, st);
        case DTYPE_BF16: return launch_kv<T, DTYPE_BF16>(p, write, grid, block, st);
        case DTYPE_F16: return launch_kv<T, DTYPE_F16>(p, write, grid, block, st);
        case DTYPE_Q8_0: return launch_kv<T, DTYPE_Q8_0>(p, write, grid, block, st);
        default: return launch_kv<T, DTYPE_Q4_0>(p, write, grid, block, st);
    }
}

int kv_call(kernel_context_t *ctx, const sapphire_kv_cache_t *cache, const sapphire_kv_args_t *a, bool write) {
    const char *who = write ? "sapphire_kv_write_device" : "sapphire_kv_read_device";
    if (!ctx || !cache || !a) {
        LOG_ERROR("%s: NULL argument", who);
        return -1;
    }
    std::lock_guard<std::recursive_mutex> lk(ctx->exec_mutex);
    if (!ctx->initialized) {
        ctx_fail(ctx, who, "context not initialized");
        return -1;
    }
    KvParams p{};
    if (!kv_layout(ctx, who, cache, &p.l)) return -1;
    const size_t size = io_size(a->dtype);
    if (!size) {
        ctx_fail(ctx, who, "k and v must be F32, BF16 or F16");
        return -1;
    }
    if (a->tokens < 0 || a->sequences < 0 || (!a->cu_tokens && a->tokens != a->sequences)) {
        ctx_fail(ctx, who, "%d tokens of %d sequences (without cu_tokens each has one)", a->tokens, a->sequences);
        return -1;
    }
    if (a->tokens == 0 || a->sequences == 0) return 0;
    if (a->table_stride <= 0) {
        ctx_fail(ctx, who, "table_stride must be positive");
        return -1;
    }
    if (!on_device(ctx, who, "pages", cache->pages) || !on_device(ctx, who, "k", a->k) || !on_device(ctx, who, "v", a->v) ||
        !on_device(ctx, who, "page_table", a->page_table) ||
        (a->cu_tokens && !on_device(ctx, who, "cu_tokens", a->cu_tokens)) ||
        (a->start && !on_device(ctx, who, "start", a->start)))
        return -1;
    const long long row = (long long)cache->kv_heads * cache->head_dim;
    p.r = {a->cu_tokens, a->start, a->page_table, a->tokens, a->sequences, a->table_stride, a->k, a->v,
           a->k_token_stride ? a->k_token_stride : row, a->k_head_stride ? a->k_head_stride : cache->head_dim,
           a->v_token_stride ? a->v_token_stride : row, a->v_head_stride ? a->v_head_stride : cache->head_dim};
    p.wide = rows_aligned(a->k, p.r.k_ts, p.r.k_hs, size) && rows_aligned(a->v, p.r.v_ts, p.r.v_hs, size);
    p.err = ctx->d_err;
    p.units = cache->head_dim / kUnit;
    AttnDevice g(ctx->device);
    const int rows = kThreads / p.units, sms = sm_count(ctx->device), heads = 2 * cache->kv_heads;
    // A block's rows are heads of one token, evenly divided where there are
    // more than rows, or heads of several tokens.  It looks its tokens up
    // first, so it takes eight batches of them behind that, while every SM
    // still gets four blocks (eight: 93 -> 96 us for 8192 + 65193 tokens);
    // fewer tokens are cut finer.
    const int steps = (heads + rows - 1) / rows;
    p.row_heads = (heads + steps - 1) / steps;
    const int token_rows = rows / p.row_heads;
    p.block_tokens = std::min(kMaxTokens, 8 * kBatch * token_rows);
    while (p.block_tokens > 1 && (a->tokens + p.block_tokens - 1) / p.block_tokens < 4 * sms) p.block_tokens = (p.block_tokens + 1) / 2;
    const dim3 grid((a->tokens + p.block_tokens - 1) / p.block_tokens);
    const dim3 block(p.units, p.row_heads * std::min(token_rows, p.block_tokens));
    const cudaError_t e = a->dtype == DTYPE_F32    ? launch_kv<float>(cache->dtype, p, write, grid, block, ctx->stream)
                          : a->dtype == DTYPE_BF16 ? launch_kv<__nv_bfloat16>(cache->dtype, p, write, grid, block, ctx->stream)
                                                   : launch_kv<__half>(cache->dtype, p, write, grid, block, ctx->stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        ctx_fail(ctx, who, "launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}

// nullptr, or why the cache's shape is not supported.
const char *kv_shape(const sapphire_kv_cache_t *c, KvLayout *l) {
    const int d = c->head_dim;
    if (d != 64 && d != 96 && d != 128 && d != 192 && d != 256) return "head_dim must be 64, 96, 128, 192 or 256";
    if (c->kv_heads <= 0 || c->kv_heads > 1024) return "kv_heads must be 1 to 1024";
    if (c->page_size <= 0 || c->page_size > 4096) return "page_size must be 1 to 4096";
    const int nb = d / 32;
    l->scale_stride = 0;
    switch (c->dtype) {
        case DTYPE_F32: l->row_bytes = 4 * d; break;
        case DTYPE_BF16:
        case DTYPE_F16: l->row_bytes = 2 * d; break;
        case DTYPE_Q8_0: l->row_bytes = d; break;
        case DTYPE_Q4_0: l->row_bytes = d / 2; break;
        default: return "the cache's type must be F32, BF16, F16, Q8_0 or Q4_0";
    }
    if (c->dtype == DTYPE_Q8_0 || c->dtype == DTYPE_Q4_0) l->scale_stride = nb <= 2 ? 2 : nb <= 4 ? 4 : 8;
    const int ps = c->page_size;
    l->v_off = ps * l->row_bytes;
    l->ks_off = 2 * ps * l->row_bytes;
    l->vs_off = l->ks_off + ps * l->scale_stride * 4;
    l->chunk_bytes = l->vs_off + ps * l->scale_stride * 4;
    l->page_bytes = (unsigned long long)l->chunk_bytes * c->kv_heads;
    l->page_size = ps;
    l->kv_heads = c->kv_heads;
    l->head_dim = d;
    return nullptr;
}

}  // namespace

bool on_device(kernel_context_t *ctx, const char *who, const char *what, const void *p) {
    int dev = -1;
    if (p && ptr_is_device(p, &dev) && dev == ctx->device) return true;
    ctx_fail(ctx, who, "%s must be device memory of the context's GPU", what);
    return false;
}

bool kv_layout(kernel_context_t *ctx, const char *who, const sapphire_kv_cache_t *c, KvLayout *l) {
    const char *why = kv_shape(c, l);
    l->pages = static_cast<uint8_t *>(c->pages);
    l->num_pages = c->num_pages;
    if (!why && c->num_pages <= 0) why = "num_pages must be positive";
    // Row offsets are kept in units of 16 bytes in 32 bits.
    if (!why && l->page_bytes * (unsigned long long)c->num_pages > (1ull << 36)) why = "the cache is above 64 GB";
    if (!why && ((uintptr_t)c->pages & 15)) why = "pages must be 16-byte aligned";
    if (!why) return true;
    ctx_fail(ctx, who, "%s", why);
    return false;
}

extern "C" SAPPHIRE_API size_t sapphire_kv_page_bytes(const sapphire_kv_cache_t *cache) {
    KvLayout l{};
    return cache && !kv_shape(cache, &l) ? (size_t)l.page_bytes : 0;
}

extern "C" SAPPHIRE_API int sapphire_kv_write_device(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                                     const sapphire_kv_args_t *args) {
    return kv_call(ctx, cache, args, true);
}

extern "C" SAPPHIRE_API int sapphire_kv_read_device(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                                    const sapphire_kv_args_t *args) {
    return kv_call(ctx, cache, args, false);
}
