// attention.cu - attention of one new token of every sequence over its pages
// (include/sapphire_attention.h): arguments, workspace and choice of kernel.
// The kernels and what bounds them are in attention_kernel.cuh.
#include <climits>
#include <cmath>
#include <cstring>

#include "attention_kernel.cuh"

namespace {

// Blocks of one launch: all that the GPU holds at a time.
int attn_blocks(kernel_context_t *ctx, const sapphire_kv_cache_t *c, int group) {
    return sm_count(ctx->device) * attn_blocks_per_sm(c->dtype, c->head_dim, attn_wide(group));
}

// Workspace: the pieces' descriptions, then two partial results a block.
size_t attn_workspace(kernel_context_t *ctx, const sapphire_kv_cache_t *c, int group) {
    const size_t blocks = attn_blocks(ctx, c, group), heads = attn_tile_heads(group);
    return blocks * (sizeof(int4) + 2 * heads * (c->head_dim + 2) * sizeof(float));
}

// The largest of any call (under 5 MB), so that the context's never grows:
// growing waits for the stream.
size_t attn_workspace_most(kernel_context_t *ctx) {
    size_t most = 0;
    for (tensor_dtype_t type : {DTYPE_F32, DTYPE_BF16, DTYPE_F16, DTYPE_Q8_0, DTYPE_Q4_0})
        for (int dim : {64, 96, 128, 192, 256})
            for (int group : {1, 8}) {
                sapphire_kv_cache_t c{};
                c.dtype = type;
                c.head_dim = dim;
                most = std::max(most, attn_workspace(ctx, &c, group));
            }
    return most;
}

}  // namespace

extern "C" SAPPHIRE_API size_t sapphire_attention_workspace_bytes(kernel_context_t *ctx,
                                                                  const sapphire_kv_cache_t *cache, int sequences,
                                                                  int heads) {
    if (!ctx || !cache || sequences < 0 || heads <= 0 || !sapphire_kv_page_bytes(cache) || heads % cache->kv_heads) return 0;
    return attn_workspace(ctx, cache, heads / cache->kv_heads);
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
    if (a->table_stride <= 0 || a->window < 0 || !std::isfinite(a->scale * kLog2e)) {
        ctx_fail(ctx, who, "table_stride must be positive, window not negative and scale finite (times log2 e too)");
        return -1;
    }
    if (!on_device(ctx, who, "pages", cache->pages) || !on_device(ctx, who, "q", a->q) ||
        !on_device(ctx, who, "out", a->out) || !on_device(ctx, who, "page_table", a->page_table) ||
        !on_device(ctx, who, "lengths", a->lengths) || (a->lse && !on_device(ctx, who, "lse", a->lse)))
        return -1;
    // The kernels number tiles (of 64 tokens or more, and what an item costs besides) in 31 bits.
    if ((double)a->sequences * a->heads * ((double)a->table_stride * cache->page_size / 64 + 1 + kAttnItemUnits) >=
        2147483648.0) {
        ctx_fail(ctx, who, "%d sequences of up to %d pages are more tiles than 2^31", a->sequences, a->table_stride);
        return -1;
    }
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
    p.scale = (a->scale != 0.0f ? a->scale : 1.0f / sqrtf((float)cache->head_dim)) * kLog2e;
    p.err = ctx->d_err;
    p.io = a->dtype;
    p.group = a->heads / cache->kv_heads;
    p.head_tiles = (p.group + attn_tile_heads(p.group) - 1) / attn_tile_heads(p.group);
    p.page_mul = (1ull << 32) / cache->page_size + 1;
    // Side by side: as many head tiles as divide their number evenly, up to 8.
    p.blocks = attn_blocks(ctx, cache, p.group);
    p.sides = std::min(std::min(p.head_tiles, 8), p.blocks);
    while (p.head_tiles % p.sides) --p.sides;
    p.blocks -= p.blocks % p.sides;
    p.side_tiles = p.head_tiles / p.sides;
    p.code[0] = 0x64006400u;
    p.code[1] = cache->dtype == DTYPE_Q8_0 ? 0x64806480u : 0x64086408u;
    p.code[2] = 0x2c002c00u;
    p.code[3] = 0xd480d480u;
    p.aligned = cache->page_size % 16 == 0;
    p.device = ctx->device;
    const long long items = (long long)a->sequences * cache->kv_heads * p.head_tiles;
    p.by_item = items <= p.blocks;
    p.joins = (int)std::min<long long>(items, p.blocks);
    // Blocks to an item: on average, and at most one for each tile that the table
    // or the window leaves it.  (The average says nothing of one sequence far longer
    // than the others: 131072 tokens of Q8_0 beside 31 of 500, one KV head, 45 us
    // where the last block joins, 27 where the other kernel does.)
    const int tile = 16 * kAttnWarps * attn_m_tiles(cache->dtype, cache->head_dim);
    const long long room = std::min((long long)a->table_stride * cache->page_size, a->window ? (long long)a->window + tile : INT_MAX);
    p.few_holders = p.blocks <= 16 * items || (room + tile - 1) / tile <= 16;
    AttnDevice g(ctx->device);
    const size_t need = attn_workspace(ctx, cache, p.group);
    char *ws = static_cast<char *>(a->workspace);
    if (ws) {
        if (a->workspace_bytes < need || ((uintptr_t)ws & 15)) {
            ctx_fail(ctx, who, "the workspace needs %zu bytes, 16-byte aligned", need);
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
        // The context's own begins with zeroed counters: with few blocks to an item
        // the last of them joins their pieces, which saves a launch.
        const size_t counts = ((size_t)sm_count(ctx->device) * kAttnMaxBlocks * sizeof(int) + 15) & ~(size_t)15;
        if (!ctx->d_attn && ensure_scratch(ctx, &ctx->d_attn, &ctx->d_attn_cap, counts + attn_workspace_most(ctx))) return -1;
        ws = reinterpret_cast<char *>(ctx->d_attn) + counts;
        if (p.few_holders) p.count = reinterpret_cast<int *>(ctx->d_attn);
    }
    p.piece = reinterpret_cast<int4 *>(ws);
    p.part = reinterpret_cast<float *>(ws + (size_t)p.blocks * sizeof(int4));
    cudaError_t e;
    switch (cache->dtype) {
        case DTYPE_F32: e = attn_run_f32(p, ctx->stream); break;
        case DTYPE_BF16: e = attn_run_bf16(p, ctx->stream); break;
        case DTYPE_F16: e = attn_run_f16(p, ctx->stream); break;
        case DTYPE_Q8_0: e = attn_run_q8_0(p, ctx->stream); break;
        default: e = attn_run_q4_0(p, ctx->stream); break;
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        ctx_fail(ctx, who, "launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
