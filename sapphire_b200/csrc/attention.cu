// attention.cu - attention of one new token of every sequence over its pages
// (include/sapphire_attention.h).
//
//   out = sum_t softmax(scale q . k_t) v_t, one pass over the positions with a
//   running maximum m, sum l and unnormalised acc = sum exp(s - m) v
//
// One block per (sequence, query head): its warps take every eighth position,
// a lane owns one dimension of each 32, and the warps' (m, l, acc) are joined
// in shared memory.
#include <cmath>
#include <cstring>

#include "attention.cuh"

namespace {

constexpr int kWarps = 8;
constexpr int kMaxBlocks = 8;     // 32-value blocks of a head

struct AttnParams {
    KvLayout l;
    const void *q;
    void *out;
    float *lse;
    long long q_ss, q_hs, out_ss, out_hs;
    const int *page_table, *lengths;
    int sequences, heads, table_stride, length_offset, window;
    float scale;
    int *err;
};

// Value 32 b + lane of a row.
template <int kCache>
__device__ __forceinline__ float kv_value(const uint8_t *row, const float *scales, int nb, int b, int lane) {
    const int d = 32 * b + lane;
    if (kCache == DTYPE_F32) return reinterpret_cast<const float *>(row)[d];
    if (kCache == DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(row)[d]);
    if (kCache == DTYPE_F16) return __half2float(reinterpret_cast<const __half *>(row)[d]);
    const int word = (lane >> 2) * nb + b, j = lane & 3;
    if (kCache == DTYPE_Q8_0) return (float)((int)row[word * 4 + j] - 128) * scales[b];
    return (float)((int)((reinterpret_cast<const uint16_t *>(row)[word] >> (4 * j)) & 15) - 8) * scales[b];
}

template <typename T, int kCache>
__global__ void __launch_bounds__(kWarps * 32) attention_simple_kernel(const AttnParams p) {
    __shared__ float sm[kWarps], sl[kWarps], sacc[kWarps][32 * kMaxBlocks];
    const int h = blockIdx.x, s = blockIdx.y, kh = h / (p.heads / p.l.kv_heads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nb = p.l.head_dim / 32;
    const T *q = static_cast<const T *>(p.q) + s * p.q_ss + h * p.q_hs;
    long long n = (long long)p.lengths[s] + p.length_offset;
    const long long room = (long long)p.table_stride * p.l.page_size;
    if (n < 0 || n > room) {
        if (threadIdx.x == 0) atomicOr(p.err, kErrCache);
        n = n < 0 ? 0 : room;
    }
    const long long first = p.window > 0 && n > p.window ? n - p.window : 0;
    float x[kMaxBlocks], acc[kMaxBlocks], m = -INFINITY, l = 0.0f;
    for (int b = 0; b < kMaxBlocks; ++b) {
        x[b] = b < nb ? to_f32(q[32 * b + lane]) : 0.0f;
        acc[b] = 0.0f;
    }
    for (long long t = first + warp; t < n; t += kWarps) {
        const int page = p.page_table[s * (long long)p.table_stride + t / p.l.page_size], slot = (int)(t % p.l.page_size);
        if (page < 0 || page >= p.l.num_pages) {
            if (lane == 0) atomicOr(p.err, kErrCache);
            continue;
        }
        const uint8_t *chunk = p.l.pages + page * p.l.page_bytes + (unsigned long long)kh * p.l.chunk_bytes;
        const uint8_t *k = chunk + slot * p.l.row_bytes, *v = k + p.l.v_off;
        const float *ks = reinterpret_cast<const float *>(chunk + p.l.ks_off) + slot * p.l.scale_stride;
        const float *vs = reinterpret_cast<const float *>(chunk + p.l.vs_off) + slot * p.l.scale_stride;
        float dot = 0.0f;
        for (int b = 0; b < nb; ++b) dot = fmaf(x[b], kv_value<kCache>(k, ks, nb, b, lane), dot);
        for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        const float score = dot * p.scale, top = fmaxf(m, score), keep = m == -INFINITY ? 0.0f : expf(m - top);
        const float e = score == -INFINITY ? 0.0f : expf(score - top);
        m = top;
        l = l * keep + e;
        for (int b = 0; b < nb; ++b) acc[b] = fmaf(e, kv_value<kCache>(v, vs, nb, b, lane), acc[b] * keep);
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
    for (int b = 0; b < nb; ++b) sacc[warp][32 * b + lane] = acc[b];
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w]);
    float wt[kWarps];
    for (int w = 0; w < kWarps; ++w) {
        wt[w] = sm[w] == -INFINITY ? 0.0f : expf(sm[w] - M);
        L += sl[w] * wt[w];
    }
    T *out = static_cast<T *>(p.out) + s * p.out_ss + h * p.out_hs;
    for (int d = threadIdx.x; d < p.l.head_dim; d += blockDim.x) {
        float o = 0.0f;
        for (int w = 0; w < kWarps; ++w) o = fmaf(wt[w], sacc[w][d], o);
        out[d] = from_f32<T>(M == -INFINITY ? 0.0f : o / L);
    }
    if (p.lse && threadIdx.x == 0) p.lse[(long long)s * p.heads + h] = M == -INFINITY ? -INFINITY : M + logf(L);
}

template <typename T>
void launch_simple(tensor_dtype_t cache, const AttnParams &p, cudaStream_t st) {
    const dim3 grid(p.heads, p.sequences), block(kWarps * 32);
    switch (cache) {
        case DTYPE_F32: attention_simple_kernel<T, DTYPE_F32><<<grid, block, 0, st>>>(p); break;
        case DTYPE_BF16: attention_simple_kernel<T, DTYPE_BF16><<<grid, block, 0, st>>>(p); break;
        case DTYPE_F16: attention_simple_kernel<T, DTYPE_F16><<<grid, block, 0, st>>>(p); break;
        case DTYPE_Q8_0: attention_simple_kernel<T, DTYPE_Q8_0><<<grid, block, 0, st>>>(p); break;
        default: attention_simple_kernel<T, DTYPE_Q4_0><<<grid, block, 0, st>>>(p); break;
    }
}

}  // namespace

extern "C" SAPPHIRE_API size_t sapphire_attention_workspace_bytes(kernel_context_t *ctx,
                                                                  const sapphire_kv_cache_t *cache, int sequences,
                                                                  int heads) {
    if (!ctx || !cache || sequences < 0 || heads <= 0 || !sapphire_kv_page_bytes(cache) || heads % cache->kv_heads) return 0;
    return 16;
}

extern "C" SAPPHIRE_API int sapphire_attention_device(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                                      const sapphire_attention_args_t *a) {
    const char *who = "sapphire_attention_device";
    if (!ctx || !cache || !a) {
        LOG_ERROR("%s: NULL argument", who);
        return -1;
    }
    std::lock_guard<std::recursive_mutex> lk(ctx->exec_mutex);
    if (!ctx->initialized) {
        ctx_fail(ctx, who, "context not initialized");
        return -1;
    }
    AttnParams p{};
    if (!kv_layout(ctx, who, cache, &p.l)) return -1;
    if (!io_size(a->dtype)) {
        ctx_fail(ctx, who, "q and out must be F32, BF16 or F16");
        return -1;
    }
    if (a->heads <= 0 || a->heads % cache->kv_heads || a->heads > 65535) {
        ctx_fail(ctx, who, "%d query heads over %d KV heads", a->heads, cache->kv_heads);
        return -1;
    }
    if (a->sequences < 0 || a->sequences > 65535) {
        ctx_fail(ctx, who, "sequences must be 0 to 65535");
        return -1;
    }
    if (a->sequences == 0) return 0;
    if (a->table_stride <= 0 || a->window < 0 || !std::isfinite(a->scale)) {
        ctx_fail(ctx, who, "table_stride must be positive, window not negative and scale finite");
        return -1;
    }
    if (!on_device(ctx, who, "pages", cache->pages) || !on_device(ctx, who, "q", a->q) ||
        !on_device(ctx, who, "out", a->out) || !on_device(ctx, who, "page_table", a->page_table) ||
        !on_device(ctx, who, "lengths", a->lengths) || (a->lse && !on_device(ctx, who, "lse", a->lse)))
        return -1;
    p.q = a->q;
    p.out = a->out;
    p.lse = a->lse;
    const long long row = (long long)a->heads * cache->head_dim;
    p.q_ss = a->q_seq_stride ? a->q_seq_stride : row;
    p.q_hs = a->q_head_stride ? a->q_head_stride : cache->head_dim;
    p.out_ss = a->out_seq_stride ? a->out_seq_stride : row;
    p.out_hs = a->out_head_stride ? a->out_head_stride : cache->head_dim;
    p.page_table = a->page_table;
    p.lengths = a->lengths;
    p.sequences = a->sequences;
    p.heads = a->heads;
    p.table_stride = a->table_stride;
    p.length_offset = a->length_offset;
    p.window = a->window;
    p.scale = a->scale != 0.0f ? a->scale : 1.0f / sqrtf((float)cache->head_dim);
    p.err = ctx->d_err;
    AttnDevice g(ctx->device);
    switch (a->dtype) {
        case DTYPE_F32: launch_simple<float>(cache->dtype, p, ctx->stream); break;
        case DTYPE_BF16: launch_simple<__nv_bfloat16>(cache->dtype, p, ctx->stream); break;
        default: launch_simple<__half>(cache->dtype, p, ctx->stream); break;
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        ctx_fail(ctx, who, "launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
