// attention_shared.cu - attention of one new token of every sequence of a batch
// whose sequences begin with the same tokens (include/sapphire_attention.h):
// arguments, workspace, the choice of the prefix's kernel, and the joining of its
// pieces with what each sequence has behind it.
//
// Reading the prefix once for many rows (a KV head's query heads, of every sequence)
// leaves each of its pages' bytes to 2 flops for each, so its kernel is a matrix
// product (prefix_kernel.cuh).  Under fp32 queries it is the one-token kernel
// (attention_kernel.cuh) with every sequence's heads as query heads of one sequence:
// its tf32 parts hold what a 16-bit operand would not, and it reads the prefix again
// for every few tiles of 8 rows (as many as divide their number, up to 8).
#include <algorithm>
#include <climits>
#include <cmath>

#include "prefix_kernel.cuh"

namespace {

constexpr int kJoinWarps = 8;     // of a block

struct JoinParams {
    PrefixParams prefix;          // of the tensor core kernel
    bool tc;
    int heads;
    long long entries;            // sequences * heads
    const float *own;             // [sequences][heads][head_dim]
    const float2 *own_ml;         // [sequences][heads]
    void *out;
    float *lse;
    long long out_ss, out_hs;
    int io;
};

// Adds up means, each with its maximum and sum: the weight of one is l 2^(m - M).
// kEntryWarps warps take a sequence and query head, each every kEntryWarps-th piece with
// its loads in flight, and are joined in shared memory: few entries are bound by latency,
// the fewer steps behind one another the better (16 sequences of 32 heads of 128, 18 pieces
// each: 8.2 us with one warp, 6.0 with four), many by what a warp costs (64 sequences: 10.5
// and 14 us).
template <int HD, int kEntryWarps>
__global__ void __launch_bounds__(kJoinWarps * 32) shared_join_kernel(const JoinParams p) {
    // A lane has four dims, or eight of 192 and 256.
    constexpr int kLanes = HD <= 128 ? HD / 4 : HD / 8, NB = HD / kLanes / 4, kBatch = 8 / NB;
    __shared__ float4 means[kJoinWarps][NB][32];
    __shared__ float sums[kJoinWarps], tops[kJoinWarps];
    const int warp = threadIdx.x >> 5, part = warp % kEntryWarps, lane = threadIdx.x & 31, at = 4 * min(lane, kLanes - 1);
    const long long entry = (long long)blockIdx.x * (kJoinWarps / kEntryWarps) + warp / kEntryWarps;
    const bool there = entry < p.entries;
    pdl_wait();
    const PrefixParams &f = p.prefix;
    const int s = (int)(entry / p.heads), h = (int)(entry - (long long)s * p.heads), kh = h / f.group;
    const int row = s * f.group + h - kh * f.group;
    // The pieces: of consecutive slots, `stride` means apart.
    int n = 1;
    long long first = (long long)kh * f.rows + row, stride = 0;
    if (p.tc) {
        const int set_rows = f.streams * kPrefixRows, set = row / set_rows, item = kh * f.row_sets + set;
        const PrefixRanges r = prefix_ranges(f.items, (uint32_t)prefix_length(f, false), f.tile, f.blocks);
        n = 0;
        if (r.tiles > 0) {
            unsigned b0, b1;
            prefix_holders(r, item, &b0, &b1);
            n = (int)(b1 - b0) + 1;
            first = (long long)(b0 + item) * set_rows + row - set * set_rows;
            stride = set_rows;
        }
    }
    // This warp's: what lies behind the prefix (-1) for the first, and every
    // kEntryWarps-th piece.  M: their maximum, L: the sum of their weights.
    float M = -INFINITY, L = 0.0f, y[NB][4] = {};
    for (int i0 = part - 1; there && i0 < n; i0 += kBatch * kEntryWarps) {
        float4 z[kBatch][NB];
        float2 ml[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = min(i0 + k * kEntryWarps, n - 1);
            const float *from = i < 0 ? p.own + entry * HD : f.part + (first + i * stride) * HD;
            ml[k] = __ldcg(i < 0 ? p.own_ml + entry : f.part_ml + first + i * stride);
            if (i0 + k * kEntryWarps >= n) ml[k].y = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) z[k][b] = __ldcg(reinterpret_cast<const float4 *>(from + b * (HD / NB) + at));
        }
        float top = M;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) top = ml[k].y != 0.0f ? fmaxf(top, ml[k].x) : top;
        const float ref = top == -INFINITY ? 0.0f : top, keep = attn_exp2(M - ref);
        M = top;
        L *= keep;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) y[b][j] *= keep;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            // (What has no weight may be anything.)
            const float w = ml[k].y == 0.0f ? 0.0f : ml[k].y != ml[k].y ? ml[k].y : ml[k].y * attn_exp2(ml[k].x - ref);
            L += w;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float x[4] = {z[k][b].x, z[k][b].y, z[k][b].z, z[k][b].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) y[b][j] = fmaf(w, w == 0.0f ? 0.0f : x[j], y[b][j]);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) means[warp][b][lane] = make_float4(y[b][0], y[b][1], y[b][2], y[b][3]);
    if (lane == 0) {
        tops[warp] = M;
        sums[warp] = L;
    }
    __syncthreads();
    if (part || !there) return;
    float all = -INFINITY;
#pragma unroll
    for (int k = 0; k < kEntryWarps; ++k) all = fmaxf(all, tops[warp + k]);
    const float ref = all == -INFINITY ? 0.0f : all;
    L = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) y[b][j] = 0.0f;
#pragma unroll
    for (int k = 0; k < kEntryWarps; ++k) {
        const float sum = sums[warp + k], w = sum != sum ? sum : attn_exp2(tops[warp + k] - ref);
        L = fmaf(w, sum, L);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float4 x = means[warp + k][b][lane];
            y[b][0] = fmaf(w, x.x, y[b][0]);
            y[b][1] = fmaf(w, x.y, y[b][1]);
            y[b][2] = fmaf(w, x.z, y[b][2]);
            y[b][3] = fmaf(w, x.w, y[b][3]);
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (p.lse && lane == 0) p.lse[entry] = L == 0.0f ? -INFINITY : (all + log2f(L)) * 0.6931471805599453f;
    if (lane >= kLanes) return;
    const long long to = s * p.out_ss + (long long)h * p.out_hs + at;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long o = to + b * (HD / NB) + j;
            const float v = y[b][j] * inv;
            if (p.io == DTYPE_F32) static_cast<float *>(p.out)[o] = v;
            else if (p.io == DTYPE_BF16) static_cast<__nv_bfloat16 *>(p.out)[o] = __float2bfloat16_rn(v);
            else static_cast<__half *>(p.out)[o] = __float2half_rn(v);
        }
}

template <int HD>
cudaError_t run_join(const JoinParams &p, int sms, cudaStream_t st) {
    // One warp to an entry where that fills the GPU.
    const dim3 block(kJoinWarps * 32);
    if (p.entries >= 8ll * sms)
        return launch_pdl(shared_join_kernel<HD, 1>, dim3((unsigned)((p.entries + kJoinWarps - 1) / kJoinWarps)), block, 0, st, p);
    constexpr int kEntries = kJoinWarps / 4;
    return launch_pdl(shared_join_kernel<HD, 4>, dim3((unsigned)((p.entries + kEntries - 1) / kEntries)), block, 0, st, p);
}
cudaError_t run_join(const JoinParams &p, int head_dim, int sms, cudaStream_t st) {
    switch (head_dim) {
        case 64: return run_join<64>(p, sms, st);
        case 96: return run_join<96>(p, sms, st);
        case 128: return run_join<128>(p, sms, st);
        case 192: return run_join<192>(p, sms, st);
        default: return run_join<256>(p, sms, st);
    }
}

cudaError_t run_prefix(int dtype, const PrefixParams &p, cudaStream_t st) {
    switch (dtype) {
        case DTYPE_F32: return prefix_run_f32(p, st);
        case DTYPE_BF16: return prefix_run_bf16(p, st);
        case DTYPE_F16: return prefix_run_f16(p, st);
        case DTYPE_Q8_0: return prefix_run_q8_0(p, st);
        default: return prefix_run_q4_0(p, st);
    }
}

// Whether the prefix is a product on the tensor cores.
bool on_tensor_cores(int io) { return io != DTYPE_F32; }

// The workspace of a call, in bytes from its start.
struct SharedLayout {
    size_t own, own_ml, part, part_ml, attend, count, total;
    int streams, row_sets, items, blocks;
};
SharedLayout shared_layout(kernel_context_t *ctx, const sapphire_kv_cache_t *c, int io, int sequences, int heads) {
    SharedLayout w{};
    const int group = heads / c->kv_heads;
    const long long rows = (long long)sequences * group, entries = (long long)sequences * heads;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t from = at;
        at += (bytes + 255) & ~(size_t)255;
        return from;
    };
    w.blocks = sm_count(ctx->device);
    w.count = take((size_t)sm_count(ctx->device) * kAttnMaxBlocks * sizeof(int));
    w.own = take(entries * c->head_dim * sizeof(float));
    w.own_ml = take(entries * sizeof(float2));
    size_t means = entries, attend = attn_workspace(ctx, c->dtype, c->head_dim, group);
    if (on_tensor_cores(io)) {
        // Two tiles of rows share a pass over the prefix where there are that many.
        w.streams = rows > kPrefixRows ? prefix_streams(c->head_dim) : 1;
        w.row_sets = (int)((rows + w.streams * kPrefixRows - 1) / (w.streams * kPrefixRows));
        w.items = w.row_sets * c->kv_heads;
        means = (size_t)(w.blocks + w.items) * w.streams * kPrefixRows;
    } else {
        attend = std::max(attend, attn_workspace(ctx, c->dtype, c->head_dim, (int)rows));
    }
    w.part = take(means * c->head_dim * sizeof(float));
    w.part_ml = take(means * sizeof(float2));
    w.attend = take(attend);
    w.total = at + 256;                           // (the caller's starts on 16 bytes, results on 32)
    return w;
}

// nullptr, or why this many sequences and heads are not supported.
const char *shared_shape(const sapphire_kv_cache_t *c, int sequences, int heads) {
    if (heads <= 0 || heads % c->kv_heads || heads > 65535) return "query heads must be a multiple of the KV heads, at most 65535";
    if (sequences < 0 || sequences > 65535) return "sequences must be 0 to 65535";
    if ((long long)sequences * heads > 1 << 24) return "sequences times heads must be at most 2^24";
    return nullptr;
}

}  // namespace

extern "C" SAPPHIRE_API size_t sapphire_attention_shared_workspace_bytes(kernel_context_t *ctx,
                                                                         const sapphire_kv_cache_t *cache,
                                                                         tensor_dtype_t dtype, int sequences, int heads) {
    if (!ctx || !cache || !sapphire_kv_page_bytes(cache) || !io_size(dtype) || shared_shape(cache, sequences, heads)) return 0;
    return shared_layout(ctx, cache, dtype, std::max(sequences, 1), heads).total;
}

extern "C" SAPPHIRE_API int sapphire_attention_shared_device(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                                             const sapphire_attention_shared_args_t *a) {
    const char *who = "sapphire_attention_shared_device";
    if (!ctx || !cache || !a) {
        LOG_ERROR("%s: NULL argument", who);
        return -1;
    }
    std::lock_guard<std::recursive_mutex> lk(ctx->exec_mutex);
    if (!ctx->initialized) {
        ctx_fail(ctx, who, "context not initialized");
        return -1;
    }
    KvLayout l{};
    if (!kv_layout(ctx, who, cache, &l)) return -1;
    const size_t size = io_size(a->dtype);
    if (!size) {
        ctx_fail(ctx, who, "q and out must be F32, BF16 or F16");
        return -1;
    }
    if (const char *why = shared_shape(cache, a->sequences, a->heads)) {
        ctx_fail(ctx, who, "%s (%d sequences, %d query heads over %d KV heads)", why, a->sequences, a->heads, cache->kv_heads);
        return -1;
    }
    if (a->sequences == 0) return 0;
    if (a->table_stride <= 0 || a->prefix_pages <= 0 || !std::isfinite(a->scale * kLog2e)) {
        ctx_fail(ctx, who, "table_stride and prefix_pages must be positive and scale finite (times log2 e too)");
        return -1;
    }
    if (!on_device(ctx, who, "pages", cache->pages) || !on_device(ctx, who, "q", a->q) ||
        !on_device(ctx, who, "out", a->out) || !on_device(ctx, who, "prefix_table", a->prefix_table) ||
        !on_device(ctx, who, "prefix_length", a->prefix_length) || !on_device(ctx, who, "page_table", a->page_table) ||
        !on_device(ctx, who, "lengths", a->lengths) || (a->lse && !on_device(ctx, who, "lse", a->lse)))
        return -1;
    const long long prefix_room = (long long)a->prefix_pages * cache->page_size;
    if (!attn_numbered(a->sequences, a->heads, (long long)a->table_stride * cache->page_size) ||
        !attn_numbered(1, (long long)a->sequences * a->heads, prefix_room)) {
        ctx_fail(ctx, who, "%d sequences of up to %d pages behind %d are more tiles than 2^31", a->sequences, a->table_stride, a->prefix_pages);
        return -1;
    }
    AttnDevice g(ctx->device);
    const SharedLayout w = shared_layout(ctx, cache, a->dtype, a->sequences, a->heads);
    char *ws = static_cast<char *>(a->workspace);
    if (ws) {
        if (a->workspace_bytes < w.total || ((uintptr_t)ws & 15)) {
            ctx_fail(ctx, who, "the workspace needs %zu bytes, 16-byte aligned", w.total);
            return -1;
        }
        if (!on_device(ctx, who, "workspace", ws)) return -1;
    } else {
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(ctx->stream, &capturing) != cudaSuccess || capturing != cudaStreamCaptureStatusNone) {
            cudaGetLastError();
            ctx_fail(ctx, who, "a captured call needs a workspace of its own");
            return -1;
        }
        if (ensure_scratch(ctx, &ctx->d_shared, &ctx->d_shared_cap, w.total)) return -1;
        ws = reinterpret_cast<char *>(ctx->d_shared);
    }

    ws = reinterpret_cast<char *>(((uintptr_t)ws + 255) & ~(uintptr_t)255);

    const int group = a->heads / cache->kv_heads, rows = a->sequences * group;
    const float scale = (a->scale != 0.0f ? a->scale : 1.0f / sqrtf((float)cache->head_dim)) * kLog2e;
    AttnParams own{};
    own.l = l;
    own.q = a->q;
    own.out = ws + w.own;
    own.ml = reinterpret_cast<float2 *>(ws + w.own_ml);
    own.q_ss = a->q_seq_stride ? a->q_seq_stride : (long long)a->heads * cache->head_dim;
    own.q_hs = a->q_head_stride ? a->q_head_stride : cache->head_dim;
    own.out_ss = (long long)a->heads * cache->head_dim;
    own.out_hs = cache->head_dim;
    own.page_table = a->page_table;
    own.lengths = a->lengths;
    own.sequences = a->sequences;
    own.heads = a->heads;
    own.table_stride = a->table_stride;
    own.table_ss = a->table_stride;
    own.length_offset = a->length_offset;
    own.scale = scale;
    own.io = a->dtype;
    own.out_io = DTYPE_F32;

    JoinParams j{};
    PrefixParams &f = j.prefix;
    f.l = l;
    f.q = a->q;
    f.q_ss = own.q_ss;
    f.q_hs = own.q_hs;
    f.table = a->prefix_table;
    f.length = a->prefix_length;
    f.table_pages = a->prefix_pages;
    f.io = a->dtype;
    f.rows = rows;
    f.group = group;
    f.scale = scale;
    f.part = reinterpret_cast<float *>(ws + w.part);
    f.part_ml = reinterpret_cast<float2 *>(ws + w.part_ml);
    f.err = ctx->d_err;
    f.device = ctx->device;
    f.unarmed = test_tc_unarmed();
    j.tc = on_tensor_cores(a->dtype);
    j.heads = a->heads;
    j.entries = (long long)a->sequences * a->heads;
    j.own = reinterpret_cast<const float *>(ws + w.own);
    j.own_ml = own.ml;
    j.out = a->out;
    j.lse = a->lse;
    j.out_ss = a->out_seq_stride ? a->out_seq_stride : (long long)a->heads * cache->head_dim;
    j.out_hs = a->out_head_stride ? a->out_head_stride : cache->head_dim;
    j.io = a->dtype;
    cudaError_t e;
    if (j.tc) {
        f.streams = w.streams;
        f.row_sets = w.row_sets;
        f.items = w.items;
        f.blocks = w.blocks;
        f.tile = prefix_tile(cache->head_dim, cache->dtype);
        f.page_mul = (1ull << 32) / cache->page_size + 1;
        // (Copies of 16 bytes count their offsets in 32 bits.)
        f.q_wide = rows_aligned(a->q, f.q_ss, f.q_hs, size) && f.q_ss >= 0 && f.q_hs >= 0 &&
                   ((double)f.q_ss * a->sequences + (double)f.q_hs * a->heads) * size < 6.8e10;
        f.count = reinterpret_cast<int *>(ws + w.count);
        f.counts = sm_count(ctx->device) * kAttnMaxBlocks;
        e = run_prefix(cache->dtype, f, ctx->stream);
        attn_plan(ctx, cache->dtype, &own, ws + w.attend, f.count);
    } else {
        AttnParams front = own;
        front.out = f.part;
        front.ml = f.part_ml;
        front.out_ss = 0;
        front.page_table = a->prefix_table;
        front.lengths = a->prefix_length;
        front.sequences = 1;
        front.heads = cache->kv_heads * rows;
        front.row_group = group;
        front.table_stride = a->prefix_pages;
        front.length_offset = 0;
        attn_plan(ctx, cache->dtype, &front, ws + w.attend, nullptr);
        e = attn_run(cache->dtype, front, ctx->stream);
        attn_plan(ctx, cache->dtype, &own, ws + w.attend, nullptr);
    }
    if (e == cudaSuccess) e = attn_run(cache->dtype, own, ctx->stream);
    if (e == cudaSuccess) e = run_join(j, cache->head_dim, sm_count(ctx->device), ctx->stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        ctx_fail(ctx, who, "launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
