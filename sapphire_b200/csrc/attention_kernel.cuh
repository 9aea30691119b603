// attention_kernel.cuh - one pass of attention of one new token over a paged
// cache; attention.cu plans and launches it.  Each cache type is compiled in a
// source of its own (attention_<type>.cu).
//
// Mathematics.  Per query head a running maximum m (of scores in units of
// log2 e), sum l and unnormalised acc = sum_t 2^(s_t - m + kBias) v_t; pieces
// of a sequence join by weights 2^(m_piece - m).
//
// What bounds it: every visible K and V row is read once from HBM, so the work
// is laid out to stream rows and to keep everything else off that path.  64
// sequences of 8192, 8 KV heads of 128, 4 query heads each (of 6554 GB/s; two
// GPUs): bf16 350 - 358 us, 0.92 - 0.94; Q8_0 205 - 228 us, 0.81 - 0.90; F32 397
// us at 32 sequences, 0.83 (one GPU); Q4_0 169 - 183 us, 0.56 - 0.61.  2 x 131071
// over Q4_0 with 5 query heads take 91 - 97 us, 0.53 - 0.56: DRAM is at 0.44 of
// its peak, a scheduler issues in 0.60 of the cycles and no pipe is near full (ALU
// 0.47), so it is the chain of each of a scheduler's 2.8 warps (copies, scores,
// softmax, unpacking, values) that holds it up.  Short calls are latency: one
// fp32 sequence of 577 takes 11 us, a block's chain of lengths, page table, rows and
// joining (20 k cycles: 2.5 k to its first item, 5 k to its first rows, 4 k for a
// tile, 8 k for the joins of its warps and of the blocks).
//
// Layout.  A warp takes 16 tokens at a time, or 32 where rows are short.  Scores are S^T = K Q^T and
// outputs O^T = V^T P^T with warp MMAs whose M side is the tile (16 tokens, or
// 16 dims) and whose N = 8 columns are query heads.  A 16-bit MMA gives fp32
// products of more bits from parts of the query and of the probability (high,
// low, ...), split one of two ways:
//   narrow (groups of at most 4 query heads): a head's high and low part are
//     neighbouring columns, which one lane holds together (c0 + c1), so two
//     parts cost one MMA;
//   wide: 8 heads are the columns and each part is an MMA of its own, one part
//     where it is exact (a bf16 query) or its rounding is far below the
//     output's (an fp16 probability under a bf16 output: 2^-12 against 2^-9).
// The MMAs are a few percent of the pass (a fifth over Q4_0).  tcgen05 tiles of
// 128 tokens or dims by 8 or 16 heads were not tried: their operands come from
// shared memory, so quantised rows would be written back unpacked, and K's scales
// need an accumulator for each 32 dims.  Rows come by asynchronous copies into two slots of
// a warp, K's and V's, while the other's is used, and a lane reads its fragments
// as vectors: the order of dims inside an MMA is free as long as both operands
// share it, so a lane's consecutive bytes of a row are its fragment.
//
//   K (A operand): lane (g, t) = (lane / 4, lane % 4) reads rows g and g + 8,
//     dims 8t .. 8t + 7 of each 32.
//   V (A operand, transposed): lane (g, t) reads tokens 2t, 2t + 1, 2t + 8,
//     2t + 9, dims 8g .. 8g + 7 of each 64, and pairs tokens with byte permutes.
//   P (B operand): a movmatrix of the packed (high, low) pairs.
//
// Quantised rows are kept as words of 4 codes in the order [8][nb], so the same
// lanes read consecutive bytes.  V's codes become fp16 exactly (1024 + code - 1152,
// or - 1032), and V's scale multiplies the probability, the product brought into
// fp16's range by a power of two per warp that follows the largest seen (products
// below 2^-27 of that lose bits).  Wide tiles under a bf16 output round it to fp16
// once, 2^-12 of it against the output's 2^-9, and the probability over fp16 rows
// too; a second part would cost 9 to 12 % there (2 x 131071 over Q4_0, 5 heads: 96
// -> 107 us), 0.5 to 3 % in narrow tiles, which have it.  K's codes become
// fp16 the same way, except in narrow tiles under a bf16 query: there they are
// multiplied as the integers they are by the query as 23-bit integers (three
// signed bytes in two MMAs), the sums exact, and a product with K's scale brings
// a block's sum to fp32.  A byte with its top bit turned is Q8_0's code, or 16
// times a Q4_0 code of the byte's high half, without its offset.  Query values
// down to 2^-14 of their head's largest keep all 8 of their bits, smaller ones
// are off by at most 2^-22 of it.  (Two bytes leave 2^-15 of it, which a few large
// channels of a query turn into errors above the output's rounding; they were 2
// to 4 % faster.)  A wide tile would need three MMAs; one fp16 part of the query
// is exact down to 2^-31 of the head's largest and faster (64 x 8192, 8 heads to
// a KV head of 128: Q8_0 239 -> 230 us, Q4_0 198 -> 187).
//
// Split.  The tiles (64 tokens of one KV head and up to 8 query heads) of all
// sequences are numbered in a row and cut into as many equal ranges as the GPU
// holds blocks (of one side, below), whatever the lengths; a block's pieces that
// do not hold a whole sequence go to the workspace.  The last of an item's blocks
// adds them up in their order, or, where an item may have many blocks or the
// workspace is the caller's (no zeroed counters), attend_join_kernel does.
#pragma once

#include "attention.cuh"

constexpr int kAttnWarps = 4;
// Shared memory of one of an SM's `blocks` blocks (each costs 1 KB besides).
constexpr int attn_smem(int blocks) { return 228 * 1024 / blocks - 1024; }
constexpr float kLog2e = 1.4426950408889634f;

// What an item costs besides its tiles (its query, the filling of the slots and
// the joining of the warps), in tiles: the ranges of blocks are cut in these
// units, so one that meets many short sequences takes fewer tiles.
constexpr int kAttnItemUnits = 2;
// Positions of a sequence: tokens are numbered in 31 bits, and look-ups run up to
// three times 2048 tokens ahead of a sequence's end.
constexpr long long kAttnMaxTokens = 0x7fffc000;
constexpr int kAttnMaxBlocks = 4;         // on an SM, of any variant

struct AttnParams {
    KvLayout l;
    const void *q;
    void *out;
    float *lse;
    float2 *ml;                    // or, where another pass joins: maximum (in units of log2 e) and sum of what out is the mean of
    long long q_ss, q_hs, out_ss, out_hs;
    const int *page_table, *lengths;
    int io, out_io;                // tensor_dtype_t of q and out
    int row_group;                 // 0, or the heads are row_group heads of many sequences, of each KV head in turn
    int sequences, heads, group;   // group: query heads of a KV head
    int head_tiles;                // tiles of 4 or 8 query heads of a group
    int sides, side_tiles;         // head tiles that blocks work on side by side, and one behind another
    int table_stride, length_offset, window;
    long long table_ss;            // entries from a sequence's table to the next one's
    int table_hs;                  // and from a KV head's (0: one table for all)
    float scale;                   // scores times log2 e
    unsigned long long page_mul;   // floor(2^32 / page_size) + 1
    bool aligned;                  // pages of a multiple of 16 tokens
    int device;
    int blocks;
    float *part;                   // [blocks][2][GH * (HD + 2)]
    // Items that several blocks hold: (sequence, head tile, blocks, first
    // block), by item where there are no more of them than blocks (by_item),
    // else by first block; 0 blocks where there is nothing to join.
    int4 *piece;
    bool by_item;
    int joins;                     // entries of piece
    bool few_holders;              // at most 16 blocks to an item, on average or at all
    int *count;                    // [blocks] zeros (and zeros again behind the call), or nullptr: attend_join_kernel joins
    int *err;
    unsigned code[4];              // CodeConst, where the compiler does not see constants
};

// Query heads of a tile for a group of this size.
inline bool attn_wide(int group) { return group > 4; }
inline int attn_tile_heads(int group) { return attn_wide(group) ? 8 : 4; }
// MMA tiles (16 tokens) of a warp's tile, and resident blocks per SM.
// (MMA tiles: two of short rows share a tile's overhead.  Blocks: as many as
// registers and shared memory allow; two for 512-byte rows of F32, 32 x 8192 over
// 128 dims 421 us with one, 396 with two, 8 query heads to a KV head 414 and 350,
// though one short sequence of 577 8.6 and 9.0.)
constexpr int attn_m_tiles(int cache, int hd) {
    return cache == DTYPE_Q4_0 || cache == DTYPE_Q8_0 || (hd <= 64 && cache != DTYPE_F32) ? 2 : 1;
}
constexpr int attn_blocks_per_sm(int cache, int hd, bool wide) {
    if (cache == DTYPE_F32) return hd <= 64 ? 3 : hd <= 128 ? 2 : 1;
    if (cache == DTYPE_Q4_0) return hd <= 64 ? 4 : hd <= 128 ? (wide ? 3 : 4) : 2;
    if (cache == DTYPE_Q8_0) return hd <= 64 ? 4 : hd <= 128 ? 3 : 2;
    return hd <= 128 ? 3 : 2;
}

#ifdef __CUDACC__

// K's codes are multiplied as integers under a bf16 query in narrow tiles.
template <int kCache, bool kWide, bool kExact>
constexpr bool kAttnInt = (kCache == DTYPE_Q8_0 || kCache == DTYPE_Q4_0) && !kWide && !kExact;
// 2^(p + kBias): probabilities use the upper end of fp16 over fp16 caches.
template <int kCache>
constexpr float kAttnBias = kCache == DTYPE_F16 ? 14.0f : 0.0f;

__device__ __forceinline__ float attn_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool kBf16>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
    if (kBf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The 11 leading bits of x, rounded half away from zero (the bits of a value are
// ordered like its magnitude): two cheap instructions where the conversion is
// one of a quarter of their rate.
__device__ __forceinline__ float take_tf32(float &x) {
    const float hi = __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
    x -= hi;
    return hi;
}
// d = a b on 32 signed bytes of each.
__device__ __forceinline__ void mma8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Packs (a, b) as two 16-bit values, a in the low half, rounded to nearest.
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if (kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <bool kBf16>
__device__ __forceinline__ float round16(float a) {
    if (kBf16) return __bfloat162float(__float2bfloat16_rn(a));
    return __half2float(__float2half_rn(a));
}
// The next part of x: what it rounds to, taken off x.
template <bool kBf16>
__device__ __forceinline__ float take16(float &x) {
    const float hi = round16<kBf16>(x);
    x -= hi;
    return hi;
}

// What unpacking codes keeps in registers: an instruction takes one constant.
struct CodeConst {
    uint32_t magic, sub, div, sub16;      // 1024; 1152 (Q8_0) or 1032; 1 / 16; 72, twice each
};
// Two bytes of `w` (selected by sel's low nibbles of positions 0 and 2; the
// others take magic's high byte) as fp16 integers - 128.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t w, const CodeConst &k) {
    uint32_t x, v;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(x) : "r"(w), "r"(k.magic), "n"(kSel));                     // 1024 + code
    asm("sub.f16x2 %0, %1, %2;" : "=r"(v) : "r"(x), "r"(k.sub));
    return v;
}
// Nibbles 0 and 4 (kShift = 0), or 1 and 5 (kShift = 4), of w as fp16 integers - 8.
template <int kShift>
__device__ __forceinline__ uint32_t nibbles_to_half2(uint32_t w, const CodeConst &k) {
    uint32_t x, v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w), "n"(kShift ? 0x00f000f0 : 0x000f000f), "r"(k.magic));   // (w & mask) | 1024
    if (kShift == 0) asm("sub.f16x2 %0, %1, %2;" : "=r"(v) : "r"(x), "r"(k.sub));                     // 1024 + code - 1032
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v) : "r"(x), "r"(k.div), "r"(k.sub16));            // (1024 + 16 code) / 16 - 72
    return v;
}

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// N (16 or 8) bytes from global to shared memory, on their way until copies_wait.
template <int N>
__device__ __forceinline__ void copy_bytes(uint32_t dst, const uint8_t *src) {
    if (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
// The same where ok, else zeros.
template <int N>
__device__ __forceinline__ void copy_or_zero(uint32_t dst, const uint8_t *src, bool ok) {
    if (ok) copy_bytes<N>(dst, src);
    else if (N == 16) asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(dst), "r"(0) : "memory");
    else asm volatile("st.shared.v2.u32 [%0], {%1,%1};" ::"r"(dst), "r"(0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// N bytes of shared memory at p (aligned to the largest power of two up to 16
// that divides N) as 32-bit words.
template <int N>
__device__ __forceinline__ void read_bytes(const uint8_t *p, uint32_t *w) {
    if constexpr (N % 16 == 0) {
#pragma unroll
        for (int i = 0; i < N / 16; ++i) {
            const uint4 u = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
    } else if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            const uint2 u = reinterpret_cast<const uint2 *>(p)[i];
            w[2 * i] = u.x, w[2 * i + 1] = u.y;
        }
    } else if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
    } else {
        static_assert(N % 2 == 0, "");
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const uint32_t h = reinterpret_cast<const uint16_t *>(p)[i];
            if (i % 2 == 0) w[i / 2] = h;
            else w[i / 2] |= h << 16;
        }
    }
}
template <int N>
__device__ __forceinline__ void read_scales(const uint8_t *p, float (&s)[N]) {
    constexpr int kPad = N <= 2 ? 2 : N <= 4 ? 4 : 8;
    float f[kPad];
    read_bytes<kPad * 4>(p, reinterpret_cast<uint32_t *>(f));
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = f[i];
}
#endif  // __CUDACC__

// Shapes of one variant.
template <int kCache, int HD, bool kWide>
struct AttnShape {
    static constexpr bool kQuant = kCache == DTYPE_Q8_0 || kCache == DTYPE_Q4_0;
    static constexpr bool kF32 = kCache == DTYPE_F32;
    static constexpr bool kBf16 = kCache == DTYPE_BF16;
    static constexpr int NB = HD / 32;
    static constexpr int kRowBytes = kCache == DTYPE_Q8_0 ? HD : kCache == DTYPE_Q4_0 ? HD / 2 : kF32 ? 4 * HD : 2 * HD;
    static constexpr int kScaleBytes = !kQuant ? 0 : NB <= 2 ? 8 : NB <= 4 ? 16 : 32;
    // Tokens of a warp's tile: two MMA tiles where rows are short.
    static constexpr int MT = attn_m_tiles(kCache, HD);
    static constexpr int kTok = 16 * MT;
    // A warp's two slots: the K and the V rows of a tile, each row padded off
    // the banks of its neighbours, and their scales.
    static constexpr int kStride = kRowBytes + (kF32 ? 32 : 16);
    static constexpr int kScaleOff = kTok * kStride;
    static constexpr int kSlot = kScaleOff + kTok * kScaleBytes;
    static constexpr int kBlocks = attn_blocks_per_sm(kCache, HD, kWide);
    static_assert(kBlocks <= kAttnMaxBlocks, "");
    // Query parts: rows of 8 columns, padded so that the rows of neighbouring
    // lanes fall on the other half of the banks.
    static constexpr int kQElem = kF32 ? 4 : 2;
    static constexpr int kQStride = (HD * kQElem) % 128 == 0 ? HD * kQElem + 64 : HD * kQElem;
    static constexpr int kDigitStride = HD % 128 == 96 ? HD : HD + 32;        // of a row of query bytes
};

#ifdef __CUDACC__
// The positions a sequence's new token attends to, as tiles.
struct AttnSpan {
    int first, end, tile0, tiles, units;
};
// (tiles of kTile tokens)
template <int kTile>
__device__ __forceinline__ AttnSpan attn_span(const AttnParams &p, int s, bool report) {
    long long n = (long long)__ldg(p.lengths + s) + p.length_offset;
    const long long room = min((long long)p.table_stride * p.l.page_size, kAttnMaxTokens);
    if (n < 0 || n > room) {
        if (report) atomicOr(p.err, kErrCache);
        n = n < 0 ? 0 : room;
    }
    AttnSpan a;
    a.end = (int)n;
    a.first = p.window > 0 && a.end > p.window ? a.end - p.window : 0;
    a.tile0 = a.first / kTile;
    a.tiles = max(1, (a.end + kTile - 1) / kTile - a.tile0);      // an empty sequence still writes its zeros
    a.units = a.tiles + kAttnItemUnits;
    return a;
}

// Parts of a query and of a probability, as B operands (narrow: one holds two
// parts, two hold three; wide: one part each).  kExact: fp32 and fp16 queries.
template <int kCache, bool kWide, bool kExact>
struct AttnParts {
    static constexpr int kQS = !kWide ? (kCache == DTYPE_BF16 && kExact ? 2 : 1)
                               : kCache == DTYPE_F32 ? 2 : kCache == DTYPE_BF16 ? (kExact ? 3 : 1) : kExact ? 2 : 1;
    // Three signed bytes: the low and the middle one in one MMA, the high one in another.
    static constexpr bool kInt = kAttnInt<kCache, kWide, kExact>;
    static constexpr int kSets = kInt ? 2 : kQS;                  // rows of 8 columns of the query
    static constexpr int kPS = !kWide ? kQS : kCache == DTYPE_F32 ? 2 : kCache == DTYPE_BF16 ? (kExact ? 3 : 2) : kExact ? 2 : 1;
};

// Shared memory of the query's parts.
template <int kCache, int HD, bool kWide, bool kExact>
constexpr int attn_query_bytes() {
    using Pt = AttnParts<kCache, kWide, kExact>;
    using Sh = AttnShape<kCache, HD, kWide>;
    return Pt::kSets * 8 * (Pt::kInt ? Sh::kDigitStride : Sh::kQStride);
}

// Adds holders i0, i0 + step, ... below n of head h's item to M, L and o,
// kBatch of them in flight.  part: the first one's partial; the others' follow
// as the first slots of the next blocks.
template <int HD, int kBatch>
__device__ __forceinline__ void attn_add_holders(const float *part, size_t stride, int tile_heads, int h, int i0, int step,
                                                 int n, float &M, float &L, float (&o)[HD / 32]) {
    constexpr int kVals = HD / 32;
    const int lane = threadIdx.x & 31;
    for (; i0 < n; i0 += step * kBatch) {
        float m[kBatch], l[kBatch], x[kBatch][kVals], top = M;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = i0 + k * step;
            m[k] = -INFINITY;
            l[k] = 0.0f;
            if (i >= n) {
#pragma unroll
                for (int j = 0; j < kVals; ++j) x[k][j] = 0.0f;
                continue;
            }
            const float *from = part + (i ? 2 * i - 1 : 0) * stride;
            m[k] = __ldcg(from + h);
            l[k] = __ldcg(from + tile_heads + h);
#pragma unroll
            for (int j = 0; j < kVals; ++j) x[k][j] = __ldcg(from + 2 * tile_heads + h * HD + 32 * j + lane);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) top = fmaxf(top, m[k]);
        const float ref = top == -INFINITY ? 0.0f : top, keep = attn_exp2(M - ref);
        M = top;
        L *= keep;
#pragma unroll
        for (int j = 0; j < kVals; ++j) o[j] *= keep;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float w = l[k] != l[k] ? l[k] : attn_exp2(m[k] - ref);      // a NaN's maximum says nothing
            L = fmaf(w, l[k], L);
#pragma unroll
            for (int j = 0; j < kVals; ++j) o[j] = fmaf(w, x[k][j], o[j]);
        }
    }
}
__device__ __forceinline__ void attn_store(const AttnParams &p, long long at, float y) {
    if (p.out_io == DTYPE_F32) static_cast<float *>(p.out)[at] = y;
    else if (p.out_io == DTYPE_BF16) static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(y);
    else static_cast<__half *>(p.out)[at] = __float2half_rn(y);
}

__device__ __forceinline__ void attn_store_lse(const AttnParams &p, long long at, float M, float L) {
    if (p.ml) p.ml[at] = make_float2(M, L);
    else if (p.lse) p.lse[at] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

template <int kCache, int HD, bool kWide, bool kExact>
__global__ void __launch_bounds__(kAttnWarps * 32, attn_blocks_per_sm(kCache, HD, kWide)) attend_kernel(const AttnParams p) {
    using Sh = AttnShape<kCache, HD, kWide>;
    using Pt = AttnParts<kCache, kWide, kExact>;
    constexpr int GH = kWide ? 8 : 4, HL = kWide ? 2 : 1;         // heads of a tile, and of a lane
    constexpr int NB = Sh::NB, MT = Sh::MT, kTok = Sh::kTok, kTile = kTok * kAttnWarps, kMTiles = HD / 16;
    constexpr int kQS = Pt::kQS, kPS = Pt::kPS;
    constexpr bool kInt = kAttnInt<kCache, kWide, kExact>;
    constexpr bool kBf16 = Sh::kBf16, kF32 = Sh::kF32;
    constexpr float kBias = kAttnBias<kCache>;
    extern __shared__ __align__(16) uint8_t shared[];
    uint8_t *const sq = shared;                                   // the query's parts
    uint8_t *const slots = shared + attn_query_bytes<kCache, HD, kWide, kExact>();  // [warp][2]; at the end of an item the warps'
    float *const sacc = reinterpret_cast<float *>(slots);         // outputs [warp][head][dim]
    static_assert(2 * Sh::kSlot >= GH * HD * 4, "the warps' outputs do not fit the slots");
    __shared__ float sm_m[kAttnWarps][GH], sm_l[kAttnWarps][GH];
    __shared__ float qmul[GH];
    __shared__ unsigned warp_sum[kAttnWarps];
    __shared__ int found_seq;
    __shared__ unsigned found_base;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_trigger();
    pdl_wait();

    // ---- this block's range [lo, hi) of all items' units (fewer than 2^31,
    //      checked on the host) ----
    const int per_thread = (p.sequences + kAttnWarps * 32 - 1) / (kAttnWarps * 32);
    const int s0 = min(tid * per_thread, p.sequences), s1 = min(s0 + per_thread, p.sequences);
    // The sides' blocks of one rank walk the same tokens for head tiles of their
    // own, so a row comes from HBM once and from L2 for the others (64 x 8192, 16
    // query heads to a KV head of 128: bf16 704 -> 576 us, Q8_0 454 -> 425 us
    // against one tile behind another).  An item: a KV head and one of this
    // side's head tiles.
    const int side = blockIdx.y, side_tiles = p.side_tiles, side_blocks = gridDim.x;
    const int rows = p.l.kv_heads * side_tiles;                   // items of a sequence
    unsigned mine = 0;
    for (int s = s0; s < s1; ++s) mine += attn_span<kTile>(p, s, blockIdx.x == 0 && side == 0).units;
    unsigned incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    unsigned total = 0, base = incl - mine;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
        if (w < warp) base += warp_sum[w];
        total += warp_sum[w];
    }
    base *= rows;
    total *= rows;
    const unsigned blocks = min((unsigned)side_blocks, total), bid = blockIdx.x, slot0 = side * side_blocks;
    if (bid >= blocks) {
        if (tid == 0 && !p.count && !p.by_item) p.piece[slot0 + bid] = make_int4(0, 0, 0, 0);
        return;
    }
    // The first `longer` blocks take each + 1 units, the others each.
    const unsigned each = total / blocks, longer = total - each * blocks;
    const unsigned lo = bid * each + min(bid, longer), hi = lo + each + (bid < longer ? 1 : 0);
    if (lo >= base && lo - base < mine * rows) {
        for (int s = s0; s < s1; ++s) {
            const unsigned n = (unsigned)attn_span<kTile>(p, s, false).units * rows;
            if (lo < base + n) {
                found_seq = s;
                found_base = base;
                break;
            }
            base += n;
        }
    }
    __syncthreads();
    int seq = found_seq;
    unsigned seq_base = found_base;
    int4 piece = make_int4(0, 0, 0, 0);
    const CodeConst codes = {p.code[0], p.code[1], p.code[2], p.code[3]};

    unsigned pos = lo;
    while (pos < hi) {
        AttnSpan sp = attn_span<kTile>(p, seq, false);
        if (pos - seq_base >= (unsigned)sp.units * rows) {
            seq_base += (unsigned)sp.units * rows;
            ++seq;
            continue;
        }
        const int item = (int)((pos - seq_base) / (unsigned)sp.units);
        // The item's tiles are its last units; this block takes those in its range.
        const unsigned tile_unit = seq_base + (unsigned)(item * sp.units) + kAttnItemUnits;
        const unsigned end = min(hi, tile_unit + sp.tiles);
        if (end <= tile_unit) break;                              // the next block has its first tile
        const int piece0 = pos > tile_unit ? (int)(pos - tile_unit) : 0, piece1 = (int)(end - tile_unit);
        const int kh = item / side_tiles, ht = (item - kh * side_tiles) * p.sides + side;
        const int nh = min(GH, p.group - ht * GH);                // heads of this tile
        const int head0 = kh * p.group + ht * GH;
        const uint8_t *head = p.l.pages + (unsigned long long)kh * p.l.chunk_bytes;
        const int *table = p.page_table + (long long)seq * p.table_ss + (long long)kh * p.table_hs;
        const unsigned page16 = (unsigned)(p.l.page_bytes >> 4);
        const int tile_first = sp.tile0 + piece0, tile_end = sp.tile0 + piece1;

        const bool aligned = p.aligned;

        // ---- where a tile's tokens are ----
        // Pages of a multiple of 16 tokens (aligned): an MMA tile is a run of
        // rows of one page, a group.  Lane l looks up group l % MT of tile l / MT
        // of the next 32 / MT tiles, so a look-up of the table serves many
        // tiles, and the page ids of the ones behind are on their way.  Others:
        // lane l looks up token l of a tile, a tile ahead, and the copying lanes
        // ask it.  Either gives offsets of rows and K's scales in units of 16
        // bytes from the head (scales of tokens: their page's and the slot); V's
        // lie at fixed distances.
        constexpr int kBatch = 32 / MT;                           // tiles of one look-up
        const int tok_end = min(sp.end, tile_end * kTile);
        int look_tok = tile_first * kTile + warp * kTok + (aligned ? lane / MT * kTile + lane % MT * 16 : lane);
        const int look_step = aligned ? kBatch * kTile : kTile;
        int entry, slot;
        auto fetch = [&]() {
            int pg = (int)(((unsigned long long)(unsigned)look_tok * p.page_mul) >> 32);
            slot = look_tok - pg * p.l.page_size;
            if (slot < 0) {
                --pg;
                slot += p.l.page_size;
            }
            const bool want = aligned ? look_tok + 16 > sp.first && look_tok < tok_end
                                      : lane < kTok && look_tok >= sp.first && look_tok < tok_end;
            entry = want ? __ldg(table + pg) : -1;
            look_tok += look_step;
        };
        constexpr unsigned kAll = kTok == 32 ? 0xffffffffu : 0xffffu;
        constexpr int PR = Sh::kRowBytes / 16, kCopies = kTok * PR / 32;      // pieces of a row, copies of a lane
        static_assert(kTok * PR % 32 == 0, "");
        constexpr int kPer = Sh::kScaleBytes == 32 ? 2 : 1, kPiece = Sh::kScaleBytes == 8 ? 8 : 16;       // of a token's scales
        constexpr int kScaleCopies = Sh::kQuant ? kTok * kPer / 32 : 0;
        unsigned row16 = 0, scale16 = 0, found = 0, valid = 0;
        int token_slot = 0, load_tok = tile_first * kTile + warp * kTok, tiles_found = 0;
        unsigned group16[MT], scales16[kScaleCopies > 0 ? kScaleCopies : 1];  // of the tile that is copied, aligned
        auto resolve = [&]() {
            if (!aligned || tiles_found == 0) {
                const bool ok = (unsigned)entry < (unsigned)p.l.num_pages;
                const unsigned page_at = ok ? (unsigned)entry * page16 : 0u;
                row16 = page_at + (unsigned)(slot * PR);
                scale16 = aligned ? page_at + (unsigned)(slot * Sh::kScaleBytes / 16) : page_at;
                token_slot = slot;
                found = __ballot_sync(0xffffffffu, ok);
                tiles_found = kBatch;
                fetch();
            }
            valid = found;
            if (aligned) {
                const int at = (kBatch - tiles_found) * MT;
#pragma unroll
                for (int i = 0; i < MT; ++i) group16[i] = __shfl_sync(0xffffffffu, row16, at + i);
#pragma unroll
                for (int j = 0; j < kScaleCopies; ++j)            // each lane its token's group
                    scales16[j] = __shfl_sync(0xffffffffu, scale16, at + (32 * j + lane) / kPer / 16);
                const unsigned here = (found >> at) & (MT == 2 ? 3u : 1u);
                valid = here == (MT == 2 ? 3u : 1u) ? kAll : (here & 1 ? 0xffffu : 0u) | (here & 2 ? 0xffff0000u : 0u);
                --tiles_found;
            }
            if (load_tok < sp.first || load_tok + kTok > tok_end || (aligned && valid != kAll)) {
                const int l0 = max(sp.first - load_tok, 0), l1 = min(tok_end - load_tok, kTok);
                const unsigned inside = l1 > l0 ? (0xffffffffu >> (32 - l1)) & (0xffffffffu << l0) : 0u;
                if ((valid & inside) != inside && lane == 0) atomicOr(p.err, kErrCache);
                valid &= inside;
            } else if (!aligned && valid != kAll) {
                if (lane == 0) atomicOr(p.err, kErrCache);
            }
            load_tok += kTile;
        };

        // ---- K or V rows of a tile into the warp's slots ----
        const uint8_t *const k_slot = slots + warp * 2 * Sh::kSlot, *const v_slot = k_slot + Sh::kSlot;
        const uint32_t slots_at = smem_addr(k_slot);
        const uint8_t *const k_rows = head + lane * 16, *const v_rows = k_rows + p.l.v_off;
        const uint8_t *const k_scales = head + p.l.ks_off + lane * kPiece, *const v_scales = k_scales + (p.l.vs_off - p.l.ks_off);
        // Piece 32 j + lane of the rows: its row, its place in the slot, and its
        // place in the group's run of rows.
        auto row_of = [&](int j) { return 32 % PR == 0 ? j * (32 / PR) + lane / PR : PR % 32 == 0 ? j / (PR / 32) : (32 * j + lane) / PR; };
        auto to = [&](int j) {
            const int col = 32 % PR == 0 ? lane % PR : PR % 32 == 0 ? 32 * (j % (PR / 32 > 0 ? PR / 32 : 1)) + lane : (32 * j + lane) % PR;
            return row_of(j) * Sh::kStride + col * 16;
        };
        auto copy_rows = [&](bool is_v) {
            const uint32_t dst = slots_at + (is_v ? Sh::kSlot : 0), sdst = dst + Sh::kScaleOff + lane * kPiece;
            if (!valid) {
                // nothing of this tile counts
            } else if (aligned) {
                const uint8_t *src[MT], *ssrc[kScaleCopies > 0 ? kScaleCopies : 1];
#pragma unroll
                for (int i = 0; i < MT; ++i) src[i] = (is_v ? v_rows : k_rows) + (unsigned long long)group16[i] * 16;
#pragma unroll
                for (int j = 0; j < kScaleCopies; ++j)            // lane's token of its group
                    ssrc[j] = (is_v ? v_scales : k_scales) + (unsigned long long)scales16[j] * 16 + 512 * j - (32 * j + lane) / kPer / 16 * 16 * Sh::kScaleBytes;
                auto from = [&](int j) {
                    constexpr bool kWhole = 16 * PR % 32 == 0;    // a copy lies in one group
                    const int i = kWhole ? 2 * j / PR : row_of(j) / 16;
                    return (i == 0 ? src[0] : src[MT - 1]) + (512 * j - i * 16 * Sh::kRowBytes);
                };
                if (valid == kAll) {
#pragma unroll
                    for (int j = 0; j < kCopies; ++j) copy_bytes<16>(dst + to(j), from(j));
#pragma unroll
                    for (int j = 0; j < kScaleCopies; ++j) copy_bytes<kPiece>(sdst + 512 * j, ssrc[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < kCopies; ++j) copy_or_zero<16>(dst + to(j), from(j), (valid >> row_of(j)) & 1);
#pragma unroll
                    for (int j = 0; j < kScaleCopies; ++j) copy_or_zero<kPiece>(sdst + 512 * j, ssrc[j], (valid >> ((32 * j + lane) / kPer)) & 1);
                }
            } else {
                const uint8_t *base = head + (is_v ? p.l.v_off : 0), *sbase = head + (is_v ? p.l.vs_off : p.l.ks_off);
#pragma unroll 8
                for (int j = 0; j < kCopies; ++j) {
                    const int i = 32 * j + lane, row = i / PR, col = i - row * PR;
                    const unsigned o = __shfl_sync(0xffffffffu, row16, row) + col;
                    copy_or_zero<16>(dst + row * Sh::kStride + col * 16, base + ((unsigned long long)o << 4), (valid >> row) & 1);
                }
                for (int j = 0; j < kScaleCopies; ++j) {
                    const int i = 32 * j + lane, row = i / kPer;
                    const unsigned o = __shfl_sync(0xffffffffu, scale16, row);
                    const int sl = __shfl_sync(0xffffffffu, token_slot, row);
                    copy_or_zero<kPiece>(sdst + 512 * j, sbase + ((unsigned long long)o << 4) + sl * Sh::kScaleBytes + (i - row * kPer) * kPiece, (valid >> row) & 1);
                }
            }
            copies_commit();
        };

        // ---- the first tile's rows, and the query's values ----
        fetch();
        constexpr int kPerWarp = GH / kAttnWarps;
        float x[kPerWarp][NB];
#pragma unroll
        for (int k = 0; k < kPerWarp; ++k) {
            const int j = warp + k * kAttnWarps;
            long long off = seq * p.q_ss + (long long)(head0 + j) * p.q_hs + lane;
            if (p.row_group) {
                const int row = ht * GH + j, s = row / p.row_group;
                off = s * p.q_ss + (long long)(kh * p.row_group + row - s * p.row_group) * p.q_hs + lane;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
                x[k][b] = j >= nh ? 0.0f
                          : p.io == DTYPE_F32  ? __ldg(static_cast<const float *>(p.q) + off + 32 * b)
                          : p.io == DTYPE_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p.q)[off + 32 * b])
                                               : __half2float(static_cast<const __half *>(p.q)[off + 32 * b]);
        }
        __syncthreads();                                          // the last item's readers of the slots
        resolve();
        unsigned next_counts = valid;                             // tokens of the next tile that count
        copy_rows(false);
#pragma unroll
        for (int k = 0; k < kPerWarp; ++k) {
            const int j = warp + k * kAttnWarps;
            // Scores grow with the products: a negative scale turns the query.
            float up = p.scale < 0.0f ? -1.0f : 1.0f, mul = fmaxf(fabsf(p.scale), 1.2e-38f), top = 0.0f;
            if (!kBf16 && !kF32) {
                // fp16 parts: the head's largest value goes to [2^14, 2^15).
#pragma unroll
                for (int b = 0; b < NB; ++b) top = x[k][b] == x[k][b] ? fmaxf(top, fabsf(x[k][b])) : INFINITY;
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                if (top > 0.0f && top < INFINITY) {
                    const int e = min(141 - (int)(__float_as_uint(top) >> 23), kInt ? 119 : 126);
                    up *= __uint_as_float((uint32_t)(127 + e) << 23);
                    mul = fmaxf(mul * __uint_as_float((uint32_t)(127 - e) << 23), 1.2e-38f);
                }
            }
            const int col = kWide ? j : 2 * j;
            if constexpr (kInt) {
                // 23-bit integers: the head's largest value goes to [2^21, 2^22);
                // a head with an infinity or a NaN has no score.
                if (!(top < INFINITY)) mul = __uint_as_float(0x7fc00000u);
                up *= 128.0f;
                mul *= kCache == DTYPE_Q8_0 ? 0x1p-7f : 0x1p-11f; // (Q4_0's codes come times 16)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int y = top < INFINITY ? __float2int_rn(x[k][b] * up) : 0, y1 = (y + 128) >> 8;
                    int d = 32 * b + lane;
                    if (kCache == DTYPE_Q4_0) d = (d & ~7) | ((d & 1) << 2) | ((d >> 1) & 3);   // evens, odds
                    uint8_t *to = sq + col * Sh::kDigitStride + d;
                    to[0] = (uint8_t)y;
                    to[Sh::kDigitStride] = (uint8_t)y1;
                    to[8 * Sh::kDigitStride] = (uint8_t)((y1 + 128) >> 8);
                    to[9 * Sh::kDigitStride] = 0;
                }
                if (lane == 0) qmul[j] = mul;
                continue;
            }
            if (lane == 0) qmul[j] = mul;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float y = x[k][b] * up;
                int d = 32 * b + lane;
                if (kCache == DTYPE_Q4_0) d = (d & ~7) | ((d & 3) << 1) | ((d >> 2) & 1);   // pairs (d, d + 4)
#pragma unroll
                for (int part = 0; part < (kWide ? kQS : 2 * kQS); ++part) {
                    const int set = kWide ? part : part >> 1;
                    uint8_t *to = sq + (set * 8 + col + (kWide ? 0 : part & 1)) * Sh::kQStride;
                    if (kF32) {
                        reinterpret_cast<float *>(to)[d] = take_tf32(y);
                    } else {
                        const uint32_t u = pack16<kBf16>(y, 0.0f);
                        reinterpret_cast<uint16_t *>(to)[d] = (uint16_t)u;
                        take16<kBf16>(y);
                    }
                }
            }
        }
        __syncthreads();
        copy_rows(true);                                          // behind the query's stores, which are waited for
        float qm[HL];
#pragma unroll
        for (int j = 0; j < HL; ++j) qm[j] = qmul[HL * t + j];

        // ---- the pass over this block's tiles of the item ----
        // acc: M tile of 16 dims, rows g and g + 8, of the lane's two columns.
        float acc[kMTiles][4], m[HL], l[HL];
#pragma unroll
        for (int j = 0; j < HL; ++j) {
            m[j] = -INFINITY;
            l[j] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kMTiles; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
        float vlim = 0.0f, vinv = 0.0f;                           // p times V's scale: largest that fits, and the power of two
        // Adds what an accumulator of its own holds.  An MMA truncates its sums
        // (of one sign over 2^20 tokens that is 2^-10 of them), so only a tile's
        // products share one; of a score, a few where that shows (kExact).
        auto add_up = [](float (&to)[4], const float (&c)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j] += c[j];
        };
        // While V's rows are used the next K's are on their way, and the other
        // way round.  More slots measured worse at every type and size (64 x 8192
        // over Q8_0: 210 us with two, 217 with three; over bf16 352 and 355): the
        // memory serves fewer streams faster.
        for (int tile = tile_first; tile < tile_end; ++tile) {
            copies_wait<1>();
            __syncwarp();
            const uint8_t *slot = k_slot;
            const unsigned now = next_counts;
            // ---- scores: lane (g, t) has tokens 16 i + g, + 8 of its heads ----
            float s[HL][2 * MT];
            if constexpr (Sh::kQuant) {
                constexpr int kBytes = Sh::kRowBytes / 4, kW = kBytes / 4;        // of a row in this lane
                uint32_t kr[MT][2][kW];
                float ks[MT][2][NB];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int row = 16 * i + 8 * r + g;
                        read_bytes<kBytes>(slot + row * Sh::kStride + t * kBytes, kr[i][r]);
                        read_scales<NB>(slot + Sh::kScaleOff + row * Sh::kScaleBytes, ks[i][r]);
                    }
#pragma unroll
                for (int j = 0; j < HL; ++j)
#pragma unroll
                    for (int r = 0; r < 2 * MT; ++r) s[j][r] = 0.0f;
                if constexpr (kInt) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint2 q[Pt::kSets];
#pragma unroll
                        for (int set = 0; set < Pt::kSets; ++set)
                            q[set] = *reinterpret_cast<const uint2 *>(sq + (set * 8 + g) * Sh::kDigitStride + 32 * b + 8 * t);
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            uint32_t a[4];
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                if constexpr (kCache == DTYPE_Q8_0) {
                                    a[r] = kr[i][r][b] ^ 0x80808080u;
                                    a[2 + r] = kr[i][r][NB + b] ^ 0x80808080u;
                                } else {
                                    const uint32_t u = kr[i][r][b / 2], v = kr[i][r][(NB + b) / 2];
                                    const uint32_t w = __byte_perm(u, v, (b & 1 ? 0x32 : 0x10) | ((NB + b) & 1 ? 0x7600 : 0x5400));
                                    a[r] = ((w << 4) & 0xf0f0f0f0u) ^ 0x80808080u;      // 16 (code - 8)
                                    a[2 + r] = (w & 0xf0f0f0f0u) ^ 0x80808080u;
                                }
                            }
                            int c[Pt::kSets][4];
#pragma unroll
                            for (int set = 0; set < Pt::kSets; ++set) mma8(c[set], a[0], a[1], a[2], a[3], q[set].x, q[set].y);
                            // (low and middle bytes together stay below 2^27)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const float low = (float)(c[0][2 * r] + c[0][2 * r + 1] * 256);
                                s[0][2 * i + r] = fmaf(ks[i][r][b], fmaf((float)c[1][2 * r], 65536.0f, low), s[0][2 * i + r]);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint4 q[kQS];
#pragma unroll
                        for (int set = 0; set < kQS; ++set)
                            q[set] = *reinterpret_cast<const uint4 *>(sq + (set * 8 + g) * Sh::kQStride + 64 * b + 16 * t);
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            uint32_t a[2][4];
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                if constexpr (kCache == DTYPE_Q8_0) {
#pragma unroll
                                    for (int h = 0; h < 2; ++h) {
                                        const uint32_t w = kr[i][r][h * NB + b];
                                        a[h][r] = bytes_to_half2<0x5150>(w, codes);
                                        a[h][2 + r] = bytes_to_half2<0x5352>(w, codes);
                                    }
                                } else {
                                    // halfwords b and NB + b: codes 0-3 of words 2t and 2t + 1
                                    const uint32_t u = kr[i][r][b / 2], v = kr[i][r][(NB + b) / 2];
                                    const uint32_t w = __byte_perm(u, v, (b & 1 ? 0x32 : 0x10) | ((NB + b) & 1 ? 0x7600 : 0x5400));
                                    a[0][r] = nibbles_to_half2<0>(w, codes);
                                    a[0][2 + r] = nibbles_to_half2<4>(w, codes);
                                    a[1][r] = nibbles_to_half2<0>(w >> 8, codes);
                                    a[1][2 + r] = nibbles_to_half2<4>(w >> 8, codes);
                                }
                            }
                            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int set = 0; set < kQS; ++set) {
                                mma16<false>(c, a[0][0], a[0][1], a[0][2], a[0][3], q[set].x, q[set].y);
                                mma16<false>(c, a[1][0], a[1][1], a[1][2], a[1][3], q[set].z, q[set].w);
                            }
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                if constexpr (kWide) {
                                    s[0][2 * i + r] = fmaf(ks[i][r][b], c[2 * r], s[0][2 * i + r]);
                                    s[HL - 1][2 * i + r] = fmaf(ks[i][r][b], c[2 * r + 1], s[HL - 1][2 * i + r]);
                                } else {
                                    s[0][2 * i + r] = fmaf(ks[i][r][b], c[2 * r] + c[2 * r + 1], s[0][2 * i + r]);
                                }
                            }
                        }
                    }
                }
            } else {
                float c[MT][4];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[i][j] = 0.0f;
#pragma unroll
                for (int off = 0; off < Sh::kRowBytes; off += 64) {               // 64 bytes of a row, 16 this lane's
                    uint4 q[kQS];
#pragma unroll
                    for (int set = 0; set < kQS; ++set)
                        q[set] = *reinterpret_cast<const uint4 *>(sq + (set * 8 + g) * Sh::kQStride + off + 16 * t);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        uint32_t u[4], v[4];
                        read_bytes<16>(slot + (16 * i + g) * Sh::kStride + off + 16 * t, u);
                        read_bytes<16>(slot + (16 * i + g + 8) * Sh::kStride + off + 16 * t, v);
                        float own[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        float(&to)[4] = kExact ? own : c[i];
                        uint32_t uh[4], ul[4], vh[4], vl[4];
                        if constexpr (kF32) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                float x0 = __uint_as_float(u[j]), x1 = __uint_as_float(v[j]);
                                uh[j] = __float_as_uint(take_tf32(x0));
                                vh[j] = __float_as_uint(take_tf32(x1));
                                ul[j] = __float_as_uint(x0);
                                vl[j] = __float_as_uint(x1);
                            }
                        }
#pragma unroll
                        for (int set = 0; set < kQS; ++set) {
                            if constexpr (kF32) {
                                mma_tf32(to, ul[0], vl[0], ul[1], vl[1], q[set].x, q[set].y);
                                mma_tf32(to, ul[2], vl[2], ul[3], vl[3], q[set].z, q[set].w);
                                mma_tf32(to, uh[0], vh[0], uh[1], vh[1], q[set].x, q[set].y);
                                mma_tf32(to, uh[2], vh[2], uh[3], vh[3], q[set].z, q[set].w);
                            } else {
                                mma16<kBf16>(to, u[0], v[0], u[1], v[1], q[set].x, q[set].y);
                                mma16<kBf16>(to, u[2], v[2], u[3], v[3], q[set].z, q[set].w);
                            }
                        }
                        if (kExact) add_up(c[i], own);
                    }
                }
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        if constexpr (kWide) {
                            s[0][2 * i + r] = c[i][2 * r];
                            s[HL - 1][2 * i + r] = c[i][2 * r + 1];
                        } else {
                            s[0][2 * i + r] = c[i][2 * r] + c[i][2 * r + 1];
                        }
                    }
            }
            __syncwarp();
            resolve();
            next_counts = valid;
            copy_rows(false);
            // ---- probabilities ----
            float pr[HL][2 * MT], top[HL];
            bool grew = false;
            if (now != kAll) {
#pragma unroll
                for (int j = 0; j < HL; ++j)
#pragma unroll
                    for (int r = 0; r < 2 * MT; ++r)
                        if (!((now >> (8 * r + g)) & 1)) s[j][r] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < HL; ++j) {
                top[j] = s[j][0];
#pragma unroll
                for (int r = 1; r < 2 * MT; ++r) top[j] = fmaxf(top[j], s[j][r]);
                top[j] *= qm[j];
                grew = grew || top[j] > m[j];
            }
            if (__any_sync(0xffffffffu, grew)) {
                float keep[HL];
#pragma unroll
                for (int j = 0; j < HL; ++j) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
                    const float mn = fmaxf(m[j], top[j]);
                    keep[j] = mn == -INFINITY ? 1.0f : attn_exp2(m[j] - mn);
                    m[j] = mn;
                    l[j] *= keep[j];
                }
#pragma unroll
                for (int i = 0; i < kMTiles; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] *= keep[kWide ? j & 1 : 0];
            }
#pragma unroll
            for (int j = 0; j < HL; ++j) {
                const float ref = m[j] == -INFINITY ? 0.0f : kBias - m[j];
#pragma unroll
                for (int r = 0; r < 2 * MT; ++r) {
                    pr[j][r] = now ? attn_exp2(fmaf(s[j][r], qm[j], ref)) : 0.0f;
                    l[j] += pr[j][r];
                }
            }
            // The 16-bit B operands of MMA tile i of w.
            auto operand = [&](const float (&w)[HL][2], uint32_t (&b0)[kPS], uint32_t (&b1)[kPS]) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float y[HL];
#pragma unroll
                    for (int j = 0; j < HL; ++j) y[j] = w[j][r];
#pragma unroll
                    for (int set = 0; set < kPS; ++set) {
                        uint32_t u;
                        if constexpr (kWide) {
                            u = pack16<kBf16>(y[0], y[HL - 1]);
                            if (set + 1 < kPS) {
                                take16<kBf16>(y[0]);
                                take16<kBf16>(y[HL - 1]);
                            }
                        } else {
                            const float high = take16<kBf16>(y[0]);
                            u = pack16<kBf16>(high, set == 0 ? y[0] : 0.0f);
                            if (set + 1 < kPS) take16<kBf16>(y[0]);
                        }
                        (r ? b1 : b0)[set] = transpose8x8(u);
                    }
                }
            };
            // ---- acc += V^T P^T ----
            copies_wait<1>();
            __syncwarp();
            slot = v_slot;
            if constexpr (Sh::kQuant) {
                constexpr int kBytes = Sh::kRowBytes / 8, kW = (kBytes + 3) / 4;  // of a row in this lane
                float vs[MT][2][NB], big = 0.0f;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        read_scales<NB>(slot + Sh::kScaleOff + (16 * i + 8 * r + g) * Sh::kScaleBytes, vs[i][r]);
#pragma unroll
                        for (int b = 0; b < NB; ++b) big = fmaxf(big, fabsf(vs[i][r][b]));
                    }
                // (probabilities are at most 1)
                if (__any_sync(0xffffffffu, big > vlim)) {
                    // Where a product of probability and scale is larger than
                    // fits, a new power of two brings it to [2^13, 2^14).  An
                    // infinite scale is its block's alone.
                    big = 0.0f;
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int r = 0; r < 2; ++r)
#pragma unroll
                            for (int b = 0; b < NB; ++b)
#pragma unroll
                                for (int j = 0; j < HL; ++j) {
                                    const float y = pr[j][2 * i + r] * fabsf(vs[i][r][b]);
                                    if (y < INFINITY) big = fmaxf(big, y);
                                }
#pragma unroll
                    for (int o = 16; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                    if (big > vlim) {
                        const int e = min(max((int)((__float_as_uint(big) >> 23) & 255) - 126, -100), 126);
                        const float inv = __uint_as_float((uint32_t)(141 - e) << 23);
                        const float f = vinv == 0.0f ? 0.0f : inv / vinv;
                        vinv = inv;
                        vlim = 57344.0f / inv;
#pragma unroll
                        for (int i = 0; i < kMTiles; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[i][j] *= f;
                    }
                }
#pragma unroll
                for (int j = 0; j < HL; ++j)
#pragma unroll
                    for (int r = 0; r < 2 * MT; ++r) pr[j][r] *= vinv;
                uint32_t vr[MT][4][kW];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        read_bytes<kBytes>(slot + (16 * i + 2 * t + (r & 1) + 8 * (r >> 1)) * Sh::kStride + g * kBytes, vr[i][r]);
                if (now) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        float own[2][4] = {};
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            uint32_t a[2][4];
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                if constexpr (kCache == DTYPE_Q8_0) {
                                    const uint32_t u = vr[i][2 * r][b], v = vr[i][2 * r + 1][b];
                                    const uint32_t lo2 = __byte_perm(u, v, 0x5140), hi2 = __byte_perm(u, v, 0x7362);
                                    a[0][2 * r] = bytes_to_half2<0x5150>(lo2, codes);
                                    a[0][2 * r + 1] = bytes_to_half2<0x5352>(lo2, codes);
                                    a[1][2 * r] = bytes_to_half2<0x5150>(hi2, codes);
                                    a[1][2 * r + 1] = bytes_to_half2<0x5352>(hi2, codes);
                                } else {
                                    const uint32_t w = __byte_perm(vr[i][2 * r][b / 2], vr[i][2 * r + 1][b / 2], b & 1 ? 0x7632 : 0x5410);
                                    a[0][2 * r] = nibbles_to_half2<0>(w, codes);
                                    a[0][2 * r + 1] = nibbles_to_half2<4>(w, codes);
                                    a[1][2 * r] = nibbles_to_half2<0>(w >> 8, codes);
                                    a[1][2 * r + 1] = nibbles_to_half2<4>(w >> 8, codes);
                                }
                            }
                            float w[HL][2];
#pragma unroll
                            for (int j = 0; j < HL; ++j) {
                                w[j][0] = pr[j][2 * i] * vs[i][0][b];
                                w[j][1] = pr[j][2 * i + 1] * vs[i][1][b];
                            }
                            uint32_t b0[kPS], b1[kPS];
                            operand(w, b0, b1);
#pragma unroll
                            for (int set = 0; set < kPS; ++set)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    mma16<false>(own[h], a[h][0], a[h][1], a[h][2], a[h][3], b0[set], b1[set]);
                        }
                        add_up(acc[2 * b], own[0]);
                        add_up(acc[2 * b + 1], own[1]);
                    }
                }
            } else if constexpr (kF32) {
                // 32-bit B operands: column g is head g's part (wide), or part g % 2 of head g / 2.
                static_assert(MT == 1, "");
                uint32_t pb[kPS][2][2];                               // [set][8 tokens][k = t, t + 4]
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float y[HL];
#pragma unroll
                    for (int j = 0; j < HL; ++j) y[j] = pr[j][r];
#pragma unroll
                    for (int set = 0; set < kPS; ++set) {
                        const float u = take_tf32(y[0]);
                        const float v = kWide ? take_tf32(y[HL - 1]) : y[0];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int src = (t + 4 * k) * 4 + (g >> 1);
                            const float a = __shfl_sync(0xffffffffu, u, src), b = __shfl_sync(0xffffffffu, v, src);
                            pb[set][r][k] = __float_as_uint(g & 1 ? b : a);
                        }
                    }
                }
                if (now) {
#pragma unroll
                    for (int d32 = 0; d32 < NB; ++d32) {
                        uint32_t x[4][4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) read_bytes<16>(slot + (t + 4 * r) * Sh::kStride + 128 * d32 + 16 * g, x[r]);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float own[4] = {};
#pragma unroll
                            for (int r = 0; r < 2; ++r) {             // tokens 8r .. 8r + 7
                                uint32_t h[4], lw[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    float y = __uint_as_float(x[2 * r + (k >> 1)][2 * j + (k & 1)]);
                                    h[k] = __float_as_uint(take_tf32(y));
                                    lw[k] = __float_as_uint(y);
                                }
#pragma unroll
                                for (int set = 0; set < kPS; ++set) {
                                    mma_tf32(own, lw[0], lw[1], lw[2], lw[3], pb[set][r][0], pb[set][r][1]);
                                    mma_tf32(own, h[0], h[1], h[2], h[3], pb[set][r][0], pb[set][r][1]);
                                }
                            }
                            add_up(acc[2 * d32 + j], own);
                        }
                    }
                }
            } else {
                uint32_t b0[MT][kPS], b1[MT][kPS];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    float w[HL][2];
#pragma unroll
                    for (int j = 0; j < HL; ++j) {
                        w[j][0] = pr[j][2 * i];
                        w[j][1] = pr[j][2 * i + 1];
                    }
                    operand(w, b0[i], b1[i]);
                }
                if (now) {
#pragma unroll
                    for (int off = 0; off < Sh::kRowBytes; off += 128) {
                        constexpr int kTail = Sh::kRowBytes % 128;                // 64 where the head ends
                        const int pairs = off + 128 <= Sh::kRowBytes ? 4 : 2;     // dims 2j, 2j + 1 of this lane
                        uint32_t x[MT][4][4];
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const uint8_t *row = slot + (16 * i + 2 * t + (r & 1) + 8 * (r >> 1)) * Sh::kStride + off;
                                if (kTail && off + 128 > Sh::kRowBytes) read_bytes<8>(row + 8 * g, x[i][r]);
                                else read_bytes<16>(row + 16 * g, x[i][r]);
                            }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (j >= pairs) continue;
                            float own[4] = {};
#pragma unroll
                            for (int i = 0; i < MT; ++i) {
                                const uint32_t a0 = __byte_perm(x[i][0][j], x[i][1][j], 0x5410), a1 = __byte_perm(x[i][0][j], x[i][1][j], 0x7632);
                                const uint32_t a2 = __byte_perm(x[i][2][j], x[i][3][j], 0x5410), a3 = __byte_perm(x[i][2][j], x[i][3][j], 0x7632);
#pragma unroll
                                for (int set = 0; set < kPS; ++set) mma16<kBf16>(own, a0, a1, a2, a3, b0[i][set], b1[i][set]);
                            }
                            add_up(acc[off / 32 + j], own);
                        }
                    }
                }
            }
            __syncwarp();
            copy_rows(true);
        }
        copies_wait<0>();

        // ---- join the warps ----
        const float unit = Sh::kQuant ? (vinv == 0.0f ? 0.0f : 1.0f / vinv) : 1.0f;
#pragma unroll
        for (int j = 0; j < HL; ++j) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
            if (g == 0) {
                sm_m[warp][HL * t + j] = m[j];
                sm_l[warp][HL * t + j] = l[j];
            }
        }
        __syncthreads();
        float M[HL], L[HL], f[HL];
#pragma unroll
        for (int j = 0; j < HL; ++j) {
            const int h = HL * t + j;
            M[j] = -INFINITY;
            L[j] = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) M[j] = fmaxf(M[j], sm_m[w][h]);
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) L[j] += M[j] == -INFINITY ? sm_l[w][h] : sm_l[w][h] * attn_exp2(sm_m[w][h] - M[j]);
            f[j] = M[j] == -INFINITY ? unit : unit * attn_exp2(m[j] - M[j]);
        }
#pragma unroll
        for (int i = 0; i < kMTiles; ++i) {
            // The dims of acc rows g and g + 8 of M tile i: d and d + 1.
            int d;
            if (Sh::kQuant || kF32) d = 32 * (i / 2) + 4 * g + 2 * (i & 1);
            else if ((i / 4) * 64 + 64 <= HD) d = 64 * (i / 4) + 8 * g + 2 * (i & 3);
            else d = 64 * (i / 4) + 4 * g + 2 * (i & 3);
            float2 *to = reinterpret_cast<float2 *>(sacc + (warp * GH + HL * t) * HD + d);
            if constexpr (kWide) {
                to[0] = make_float2(acc[i][0] * f[0], acc[i][2] * f[0]);
                to[HD / 2] = make_float2(acc[i][1] * f[1], acc[i][3] * f[1]);
            } else {
                to[0] = make_float2((acc[i][0] + acc[i][1]) * f[0], (acc[i][2] + acc[i][3]) * f[0]);
            }
        }
        const bool whole = piece0 == 0 && piece1 == sp.tiles;
        float *part = p.part + (size_t)(2 * (slot0 + bid) + (piece0 == 0 ? 1 : 0)) * GH * (HD + 2);
        if (warp == 0 && g == 0) {
#pragma unroll
            for (int j = 0; j < HL; ++j) {
                const int h = HL * t + j;
                if (!whole) {
                    part[h] = M[j];
                    part[GH + h] = L[j];
                } else {
                    qmul[h] = L[j] == 0.0f ? 0.0f : 1.0f / L[j];
                    if (h < nh) attn_store_lse(p, (long long)seq * p.heads + head0 + h, M[j] - kBias, L[j]);
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < GH * HD; i += kAttnWarps * 32) {
            const int h = i / HD, d = i - h * HD;
            float o = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) o += sacc[w * GH * HD + i];
            if (!whole) {
                part[2 * GH + i] = o;
            } else if (h < nh) {
                attn_store(p, seq * p.out_ss + (long long)(head0 + h) * p.out_hs + d, o * qmul[h]);
            }
        }
        // The blocks of this item: from the one that holds its first tile to the
        // one that holds its last.
        auto block_of = [&](unsigned x) {
            const unsigned split = longer * (each + 1);
            return x < split ? x / (each + 1) : longer + (x - split) / each;
        };
        if (p.count) {
            if (!whole) {
                // The one that comes last joins them, in their order.
                const unsigned first = block_of(tile_unit), holders = block_of(tile_unit + sp.tiles - 1) - first + 1;
                int *count = p.count + slot0 + first;
                __syncthreads();
                if (tid == 0) {
                    __threadfence();
                    found_seq = atomicAdd(count, 1) == (int)holders - 1;
                }
                __syncthreads();
                if (found_seq) {
                    __threadfence();
                    if (tid == 0) *count = 0;
                    const float *parts = p.part + (2 * (size_t)(slot0 + first) + 1) * GH * (HD + 2);
                    for (int h = warp; h < nh; h += kAttnWarps) {
                        float M1 = -INFINITY, L1 = 0.0f, o1[NB];
#pragma unroll
                        for (int b = 0; b < NB; ++b) o1[b] = 0.0f;
                        attn_add_holders<HD, 8>(parts, (size_t)GH * (HD + 2), GH, h, 0, 1, (int)holders, M1, L1, o1);
                        const float inv = L1 == 0.0f ? 0.0f : 1.0f / L1;
                        if (lane == 0) attn_store_lse(p, (long long)seq * p.heads + head0 + h, M1 - kBias, L1);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            attn_store(p, seq * p.out_ss + (long long)(head0 + h) * p.out_hs + 32 * b + lane, o1[b] * inv);
                    }
                }
            }
        } else if (piece0 == 0) {
            int4 mine_holds = make_int4(0, 0, 0, 0);
            if (!whole) {
                mine_holds = make_int4(seq, kh * p.head_tiles + ht, (int)(block_of(tile_unit + sp.tiles - 1) - bid) + 1, (int)(slot0 + bid));
                piece = mine_holds;
            }
            if (p.by_item && tid == 0) p.piece[(seq * p.l.kv_heads + kh) * p.head_tiles + ht] = mine_holds;
        }
        pos = end;
    }
    if (tid == 0 && !p.count && !p.by_item) p.piece[slot0 + bid] = piece;
}

// Adds up the items that several blocks hold, where the pass does not: one block
// per item and query head.  Latency bound (4 us); it does not let the next kernel start early,
// whose blocks would take the SMs before it is done (2 x 131071 over Q4_0 called
// again and again: 93 -> 112 us).  Its warps take turns at the holders, kJoinBatch of them in flight
// (maxima, sums and values together), and are joined like the blocks' warps.
template <int HD, int kJoinWarps, int kJoinBatch>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join_kernel(const AttnParams p, int tile_heads, float bias) {
    constexpr int kVals = HD / 32;
    __shared__ float so[kJoinWarps][HD], sm[kJoinWarps], sl[kJoinWarps];
    pdl_wait();
    const int4 piece = __ldcg(p.piece + blockIdx.x);
    if (piece.z == 0) return;
    const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kh = piece.y / p.head_tiles, ht = piece.y - kh * p.head_tiles;
    if (h >= min(tile_heads, p.group - ht * tile_heads)) return;
    const size_t stride = (size_t)tile_heads * (HD + 2);
    // Holder i's partial: the second slot of the first block, the first of the others.
    const float *part = p.part + (2 * (size_t)piece.w + 1) * stride;
    float M = -INFINITY, L = 0.0f, o[kVals];
#pragma unroll
    for (int j = 0; j < kVals; ++j) o[j] = 0.0f;
    attn_add_holders<HD, kJoinBatch>(part, stride, tile_heads, h, warp, kJoinWarps, piece.z, M, L, o);
#pragma unroll
    for (int j = 0; j < kVals; ++j) so[warp][32 * j + lane] = o[j];
    if (lane == 0) {
        sm[warp] = M;
        sl[warp] = L;
    }
    __syncthreads();
    float w[kJoinWarps];
    M = -INFINITY;
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) M = fmaxf(M, sm[i]);
    const float ref = M == -INFINITY ? 0.0f : M;
    L = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) {
        w[i] = sl[i] != sl[i] ? sl[i] : attn_exp2(sm[i] - ref);
        L = fmaf(w[i], sl[i], L);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int head = kh * p.group + ht * tile_heads + h;
    if (threadIdx.x == 0) attn_store_lse(p, (long long)piece.x * p.heads + head, M - bias, L);
    const long long off = piece.x * p.out_ss + (long long)head * p.out_hs;
    for (int d = threadIdx.x; d < HD; d += kJoinWarps * 32) {
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < kJoinWarps; ++i) y = fmaf(w[i], so[i][d], y);
        attn_store(p, off + d, y * inv);
    }
}

// Allows a kernel its dynamic shared memory, once on each device.
template <typename K>
cudaError_t attn_allow(K *kernel, size_t bytes, int device, std::atomic<unsigned long long> &done) {
    const unsigned long long bit = 1ull << (device & 63);
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

template <int kCache, int HD, bool kWide, bool kExact>
cudaError_t attn_launch(const AttnParams &p, cudaStream_t st) {
    using Sh = AttnShape<kCache, HD, kWide>;
    constexpr size_t kBytes = attn_query_bytes<kCache, HD, kWide, kExact>() + 2 * kAttnWarps * Sh::kSlot;
    static_assert(kBytes + 2048 <= attn_smem(Sh::kBlocks), "the rows do not fit");
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = attn_allow(attend_kernel<kCache, HD, kWide, kExact>, kBytes, p.device, done);
    if (e != cudaSuccess) return e;
    e = launch_pdl(attend_kernel<kCache, HD, kWide, kExact>, dim3(p.blocks / p.sides, p.sides), dim3(kAttnWarps * 32), kBytes, st, p);
    if (e != cudaSuccess || p.count) return e;
    // Items of few holders take small blocks, many at a time; items of many are
    // few, and want their holders in one or two rounds (2 x 36238 tokens of one
    // KV head, 220 holders each: 17.9 -> 15.9 us; 512 items of two with the large
    // blocks: 165 -> 183 us).
    constexpr int GH = kWide ? 8 : 4;
    const dim3 joins(p.joins, std::min(GH, p.group));
    if (p.few_holders) return launch_pdl(attend_join_kernel<HD, 4, 4>, joins, dim3(4 * 32), 0, st, p, GH, kAttnBias<kCache>);
    return launch_pdl(attend_join_kernel<HD, 16, 8>, joins, dim3(16 * 32), 0, st, p, GH, kAttnBias<kCache>);
}
template <int kCache, bool kWide, bool kExact>
cudaError_t attn_launch(const AttnParams &p, cudaStream_t st) {
    switch (p.l.head_dim) {
        case 64: return attn_launch<kCache, 64, kWide, kExact>(p, st);
        case 96: return attn_launch<kCache, 96, kWide, kExact>(p, st);
        case 128: return attn_launch<kCache, 128, kWide, kExact>(p, st);
        case 192: return attn_launch<kCache, 192, kWide, kExact>(p, st);
        default: return attn_launch<kCache, 256, kWide, kExact>(p, st);
    }
}
// The variant of a cache type: narrow or wide by the group; sums of their own
// and more parts (kExact) unless query and output are bf16, whose rounding hides
// what these save.
template <int kCache>
cudaError_t attn_launch(const AttnParams &p, cudaStream_t st) {
    if constexpr (kCache != DTYPE_F32) {
        if (p.io == DTYPE_BF16)
            return attn_wide(p.group) ? attn_launch<kCache, true, false>(p, st) : attn_launch<kCache, false, false>(p, st);
    }
    return attn_wide(p.group) ? attn_launch<kCache, true, true>(p, st) : attn_launch<kCache, false, true>(p, st);
}
#endif

// Workspace of a call of this shape; how it is laid out and its tiles are shared,
// from the fields that describe the call; its launches.  (attention.cu)
size_t attn_workspace(kernel_context_t *ctx, int dtype, int head_dim, int group);
void attn_plan(kernel_context_t *ctx, int dtype, AttnParams *p, char *workspace, int *count);
cudaError_t attn_run(int dtype, const AttnParams &p, cudaStream_t st);
// Whether the tiles of a call can be numbered.
bool attn_numbered(long long sequences, long long heads, long long tokens);

// One cache type each (attention_<type>.cu).
cudaError_t attn_run_f32(const AttnParams &p, cudaStream_t st);
cudaError_t attn_run_bf16(const AttnParams &p, cudaStream_t st);
cudaError_t attn_run_f16(const AttnParams &p, cudaStream_t st);
cudaError_t attn_run_q8_0(const AttnParams &p, cudaStream_t st);
cudaError_t attn_run_q4_0(const AttnParams &p, cudaStream_t st);
