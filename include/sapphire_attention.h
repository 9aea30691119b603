/*
 * sapphire_attention.h - rotary positions, a paged key-value cache and the
 * attention of one new token over it.
 *
 * The operators a serving loop puts between the library's projections: the
 * query and key heads are rotated (sapphire_rope_device), the new keys and
 * values are stored in a paged cache, as they are or quantised
 * (sapphire_kv_write_device), and every sequence's new token attends to its
 * pages (sapphire_attention_device); whole sequences come back dense with
 * sapphire_kv_read_device.  The reference does these steps on the host for one
 * sequence and a contiguous fp32 cache (src/transformer/rope.c:65-80,
 * src/transformer/attention.c:93-163, 292-309); it has no paged or quantised
 * cache, so nothing here replaces a reference function.
 *
 * All data pointers are device memory of the context's GPU, all work is
 * enqueued on the context stream and the calls return without waiting, like
 * kernel_gemv_device.  Return convention: 0 on success, -1 on error (details
 * via kernel_ctx_last_error).  What only the device can see - a page number, a
 * position or a length outside the cache - is skipped there and returned as -1
 * by the next kernel_ctx_synchronize, or by a call before it that waits for its
 * own result (kernel_gemv, a decoder).  Strides are in elements; a stride of 0
 * means contiguous ([tokens, heads, head_dim], the last dimension always
 * contiguous).  No call allocates device memory except the first attention on
 * a context without a workspace of the caller's (once, for calls of any shape).
 */
#ifndef SAPPHIRE_ATTENTION_H
#define SAPPHIRE_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#include "kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------- *
 * Rotary positions.  Pair i of a head (i < rot_dim / 2) turns by
 * position * f_i, f_i = theta^(-2i / rot_dim), scaled for long contexts:
 *   LINEAR  f / factor
 *   BANDED  by the turns r = original_context * f / 2pi a pair makes over the
 *           original context: f where r >= turns_fast, f / factor where
 *           r <= turns_slow, and (1 - s) f / factor + s f between them,
 *           s = (r - turns_slow) / (turns_fast - turns_slow)
 *   YARN    with c(r) = rot_dim ln(original_context / 2pi r) / (2 ln theta),
 *           lo = max(floor c(turns_fast), 0), hi = min(ceil c(turns_slow),
 *           rot_dim - 1), g = clamp((i - lo) / max(hi - lo, 0.001), 0, 1):
 *           (1 - g) f + g f / factor; cos and sin times attention_factor
 * Angles are within 2^-25 of a turn (that of fp32 half turns) at any 32-bit position.
 * ------------------------------------------------------------------------- */
typedef enum {
    SAPPHIRE_ROPE_HALF = 0,         /* pairs (i, i + rot_dim / 2) */
    SAPPHIRE_ROPE_INTERLEAVED = 1   /* pairs (2i, 2i + 1) */
} sapphire_rope_layout_t;

typedef enum {
    SAPPHIRE_ROPE_UNSCALED = 0,
    SAPPHIRE_ROPE_LINEAR = 1,
    SAPPHIRE_ROPE_BANDED = 2,
    SAPPHIRE_ROPE_YARN = 3
} sapphire_rope_scaling_t;

typedef struct {
    int head_dim;            /* even, at most 512 */
    int rot_dim;             /* the first rot_dim values of a head turn, the rest is copied; even; 0: head_dim */
    int layout;              /* sapphire_rope_layout_t */
    int scaling;             /* sapphire_rope_scaling_t */
    double theta;
    double factor;           /* >= 1 (LINEAR, BANDED, YARN) */
    int original_context;    /* BANDED, YARN */
    double turns_slow;       /* 0: 1 */
    double turns_fast;       /* 0: 4 (BANDED), 32 (YARN) */
    double attention_factor; /* 0: 1, and 0.1 ln(factor) + 1 for YARN */
} sapphire_rope_config_t;

typedef struct sapphire_rope sapphire_rope_t;

/** A rotation plan (its frequencies, on the context's GPU).  NULL on error.
 *  Destroy it before its context. */
SAPPHIRE_API sapphire_rope_t *sapphire_rope_create(kernel_context_t *ctx, const sapphire_rope_config_t *cfg);
SAPPHIRE_API void sapphire_rope_destroy(sapphire_rope_t *rope);

typedef struct {
    tensor_dtype_t dtype;    /* F32, BF16 or F16, of q, k and their outputs */
    int tokens;
    const int *positions;    /* [tokens] */
    /* [tokens, q_heads, head_dim]; q_heads 0: none.  q_out is q (same strides) or does not overlap it. */
    const void *q;
    void *q_out;
    int q_heads;
    long long q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride;
    const void *k;
    void *k_out;
    int k_heads;
    long long k_token_stride, k_head_stride, k_out_token_stride, k_out_head_stride;
    int inverse;             /* != 0: turn by the negative angles, cos and sin still times
                                attention_factor: the gradient of the turn */
} sapphire_rope_args_t;

SAPPHIRE_API int sapphire_rope_device(sapphire_rope_t *rope, const sapphire_rope_args_t *args);

/* ------------------------------------------------------------------------- *
 * Paged key-value cache.  The memory is the caller's: num_pages pages of
 * sapphire_kv_page_bytes each, back to back.  A page holds page_size token
 * slots of every KV head; its bytes are, for each KV head,
 *     K rows [page_size], V rows [page_size], K scales [page_size], V scales [page_size].
 * Dense formats (F32, BF16, F16): a row is head_dim values, no scales.
 * Quantised formats: a row is nb = head_dim / 32 blocks of 32 codes, by the
 * formulas of kernel_quantize_q8_0 / _q4_0; Q8_0 stores code + 128 in a byte,
 * Q4_0 four bits, low nibble first.  The codes are kept as 8 nb words of four
 * (dims 32 b + 4 w .. + 3 of block b are word w) in the order [8][nb], so the
 * lanes that multiply them read whole vectors; a row's nb fp32 scales are
 * padded to 2, 4 or 8.  Position p of a sequence is slot p % page_size of page
 * page_table[p / page_size]; pages may be shared between sequences that only
 * read them.
 * ------------------------------------------------------------------------- */
typedef struct {
    tensor_dtype_t dtype;    /* F32, BF16, F16, Q8_0 or Q4_0 */
    int page_size;           /* 1 .. 4096 */
    int kv_heads;
    int head_dim;            /* 64, 96, 128, 192 or 256 */
    int num_pages;
    void *pages;             /* 16-byte aligned, at most 64 GB */
} sapphire_kv_cache_t;

/** Bytes of one page, 0 when the shape is not supported (pages, num_pages unused). */
SAPPHIRE_API size_t sapphire_kv_page_bytes(const sapphire_kv_cache_t *cache);

/* Tokens of ragged sequences: token j of sequence s is row cu_tokens[s] + j of
 * k and v and has position start[s] + j.  Rows from cu_tokens[sequences] on
 * belong to no sequence and are left alone. */
typedef struct {
    tensor_dtype_t dtype;    /* F32, BF16 or F16, of k and v */
    int tokens;              /* rows of k and v */
    int sequences;
    const int *cu_tokens;    /* [sequences + 1]; NULL: one token each (tokens == sequences) */
    const int *start;        /* [sequences]; NULL: 0 */
    const int *page_table;   /* [sequences, table_stride] */
    int table_stride;        /* pages a sequence can have */
    void *k, *v;             /* [tokens, kv_heads, head_dim]; only read by sapphire_kv_write_device */
    long long k_token_stride, k_head_stride, v_token_stride, v_head_stride;
} sapphire_kv_args_t;

/** Store k and v in the cache (converted or quantised).  The pages a call
 *  writes belong to one sequence each. */
SAPPHIRE_API int sapphire_kv_write_device(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                          const sapphire_kv_args_t *args);
/** Read positions start[s] .. back into k and v, dequantised in fp32 and rounded once. */
SAPPHIRE_API int sapphire_kv_read_device(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                         const sapphire_kv_args_t *args);

/* ------------------------------------------------------------------------- *
 * Attention of one new token.  Sequence s has n = lengths[s] + length_offset
 * tokens in the cache (its new one among them) and attends to positions
 * max(0, n - window) .. n - 1 (window 0: all).  Query head h uses KV head
 * h / (heads / kv_heads).  out = sum_t softmax(scale q . k_t) v_t; a sequence
 * with no position to attend to gets zeros, and -inf in lse.  What lies in
 * slots that are not attended to (NaN included) has no effect.  A NaN or an
 * infinity that is attended to makes the outputs it enters NaN or infinite
 * (an infinity may come out as NaN) and no others; a head whose every score is
 * -inf gets zeros.  A finite fp32 value from 2^128 (1 - 2^-9) on may count as
 * infinite.  A length below 0 counts as
 * 0, one beyond the table (or 2^31 - 16384) as that end, and a token on a page
 * outside the cache does not count; each is an error at the next
 * kernel_ctx_synchronize.
 * The same call gives the same bits.
 * ------------------------------------------------------------------------- */
typedef struct {
    tensor_dtype_t dtype;    /* F32, BF16 or F16, of q and out */
    int sequences;
    int heads;               /* a multiple of kv_heads */
    const void *q;           /* [sequences, heads, head_dim] */
    void *out;               /* the same, not overlapping q */
    long long q_seq_stride, q_head_stride, out_seq_stride, out_head_stride;
    float *lse;              /* [sequences, heads] log of the softmax's sum, or NULL */
    const int *page_table;   /* [sequences, table_stride] */
    int table_stride;
    const int *lengths;      /* [sequences] */
    int length_offset;
    int window;
    float scale;             /* 0: 1 / sqrt(head_dim); finite, times log2 e too */
    /* sapphire_attention_workspace_bytes of device memory, 16-byte aligned,
     * that no other call uses at the same time; its contents do not matter.
     * NULL: the context's own (allocated by the first call that needs it).  A call
     * captured into a graph keeps its workspace, so it has to bring one. */
    void *workspace;
    size_t workspace_bytes;
} sapphire_attention_args_t;

/** Workspace of one call, whatever the lengths; 0 when the shape is not supported. */
SAPPHIRE_API size_t sapphire_attention_workspace_bytes(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                                       int sequences, int heads);
SAPPHIRE_API int sapphire_attention_device(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                           const sapphire_attention_args_t *args);

#ifdef __cplusplus
}
#endif

#endif /* SAPPHIRE_ATTENTION_H */
