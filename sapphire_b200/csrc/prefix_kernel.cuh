// prefix_kernel.cuh - attention of a whole batch's new tokens to a prefix that all
// of its sequences share, on the tensor cores (tcgen05); attention_shared.cu plans
// and launches it.  Each cache type is compiled in a source of its own.
//
// Mathematics.  The rows of a KV head are the query heads it serves, of every
// sequence: S = Q K^T over the prefix, P = 2^(S - m), O = P V, with a running
// maximum m and sum l a row.  A piece of the prefix leaves O / l, m and l, which
// shared_join_kernel adds up with the other pieces and with what each sequence has
// behind the prefix.
//
// What bounds it.  One pass over K and V serves up to 256 rows (two tiles of 128), so
// up to about 250 rows a KV head it is HBM by the count (4 bytes a token, dim and KV
// head in bf16 against 4 rows flops), and above that the tensor cores and the
// exponentials: a tile of 128 rows by 128 tokens of 128 dims is 1024 cycles of MMA
// and 1024 of ex2.  Measured, 64 sequences of 32 query heads on 8 KV heads of 128
// behind 32768 tokens in bf16: 49 us for 134 MB (20 at HBM's rate) and 34 GFLOP, tensor
// pipe 33 %, ex2 34 %, issue 35 %.  A block takes 80 tokens of both tiles of rows in
// about 2650 cycles: a softmax of 1500, of which 1280 are ex2's for the two tiles
// together, then the chain of P's store, O's MMAs, S's of the next tile and their load,
// which the two tiles of rows fill for each other in part only; and 8 to 9 thousand
// cycles pass before the first tile, most of them instructions that come from memory for
// the first time.  Quantised: 24 sequences of 40 heads on 8, 60001 tokens of Q4_0,
// 88 us (tensor pipe 16 %, issue 51 %): the converting warps are what the MMAs wait for.
//
// Layout.  A block per SM, whose roles are warps:
//   0 - 3, 4 - 7  softmax of the first and the second tile of rows: a thread has a
//                 row, as tensor memory does
//   8, 9          issue the MMAs of the first and the second tile of rows
//   10            hands copied rows over to them (11 only lends its registers)
//   12 - 15 (19)  bring rows into shared memory: K and V tiles in a ring of slots,
//                 [64 dims][tokens][128 bytes] with the 128-byte swizzle, which is
//                 K-major for S and N-major for O, so V needs no transposing
// Launched with 96 registers a thread (128 of 16 warps); the softmax takes 152 (168: a
// row's scores are in registers), the MMAs' warps leave 48 (88) and the others 64 (88):
// 256 * 152 + 128 * 48 + 256 * 64 = 640 * 96 (256 * 168 + 256 * 88 = 512 * 128).
// Tensor memory holds, for each tile of rows, O, S (one column a token) and P (16-bit
// pairs, the A operand of O's MMAs) in columns of their own, so S of the next tile runs
// under O of this one.  Where there are two tiles of rows each has its softmax, its MMAs'
// warp and its barriers, and they share only the slots of K and V.  Pages are of any
// size, so rows come by 16-byte copies from wherever they lie.
//
// An MMA is issued by a whole warp with the lane elected inside the instruction's own
// asm block: 33 to 64 cycles each, against 70 to 115 from a branch that one lane takes.
// Dropped, as none gained: a polynomial for part of the exponentials, the two tiles
// of rows started half a turn apart, a turn over nothing before the first tile.
//
// Rounding.  Operands are bf16 over bf16 caches under bf16 queries, else fp16:
//   a query of bf16 is brought to [2^14, 2^15) by a power of two a row, exact down to
//   2^-29 of its largest value;
//   Q8_0 and Q4_0 values are products of fp16 (their scale is rounded to it, and the
//   product), F32 and BF16 values are rounded to it once; each group of tokens (a warp's,
//   6 to 16) times a power of two that brings its largest scale or value to [2^14, 2^15).
//   K's power multiplies the group's scores, V's is added to their exponent, relative to
//   the row's largest sum of score and power so far, and O carries that one: a large value
//   without weight takes no bits from what has weight;
//   probabilities are rounded to the operand type once, as the outputs are.  m may lag
//   behind the maximum by 2^8 before O is brought up to date, so fp16 probabilities
//   reach 2^15 and keep their bits down to 2^-21 of the largest.
// Sums are fp32.  An MMA truncates its sums, so O leaves tensor memory every
// kRunTokens tokens.
#pragma once

#include "attention_kernel.cuh"
#include "prefix_ranges.h"
#include "tc.cuh"

constexpr int kPrefixRows = 128;                  // of a tile
constexpr int kPrefixMma = 8, kPrefixCopy = 12;    // first warps of these roles
constexpr int kConverters = 8;                    // warps that bring rows and convert them
// Rows that are operands as they are take four (eight: 53 -> 58 us, 64 sequences behind
// 32768 tokens in bf16).
constexpr bool prefix_raw(int cache, bool bf16) { return cache == DTYPE_F16 || (cache == DTYPE_BF16 && bf16); }
constexpr int prefix_copiers(int cache, bool bf16) { return prefix_raw(cache, bf16) ? 4 : kConverters; }
constexpr int kRunTokens = 8192;

struct PrefixParams {
    KvLayout l;
    const void *q;
    long long q_ss, q_hs;
    const int *table, *length;
    int table_pages;
    int io;                        // tensor_dtype_t of q
    int rows, group;               // rows of a KV head: sequences times group
    int streams;                   // tiles of rows side by side: 1 or 2
    int row_sets;                  // sets of `streams` tiles of a KV head
    int items;                     // kv_heads * row_sets
    int blocks;                    // of the launch
    int tile;                      // tokens of a tile
    float scale;                   // scores times log2 e
    unsigned long long page_mul;
    bool q_wide;                   // rows of q on 16 bytes
    float *part;                   // [slots][streams * 128][head_dim]
    float2 *part_ml;               // [slots][streams * 128]
    int *count;                    // of the call behind it, to be zeroed
    int counts;
    int *err;
    int device;
    int unarmed;                   // test hook: which arrival the first block withholds
};

// Tiles of rows side by side, and tokens of a tile: S, P (half as many columns) and
// O of each tile of rows share tensor memory's 512 columns, and K and V tiles what
// shared memory the queries leave.
constexpr int prefix_streams(int hd) { return hd <= 128 ? 2 : 1; }
constexpr bool prefix_quant(int cache) { return cache == DTYPE_Q8_0 || cache == DTYPE_Q4_0; }
constexpr int prefix_tile(int hd, int cache) { return hd <= 64 ? 128 : hd <= 96 ? 96 : hd <= 192 ? 80 : prefix_quant(cache) ? 48 : 64; }
constexpr int prefix_chunks(int hd) { return (hd + 63) / 64; }
constexpr int prefix_query_bytes(int hd) { return prefix_chunks(hd) * kPrefixRows * 128; }
constexpr int prefix_slot_bytes(int hd, int cache) { return prefix_chunks(hd) * prefix_tile(hd, cache) * 128; }
constexpr int kPrefixShared = 217 * 1024;
constexpr int prefix_slots(int hd, int cache) {
    const int most = prefix_quant(cache) ? (hd <= 128 ? 4 : 3) : 8;
    const int n = (kPrefixShared - prefix_streams(hd) * prefix_query_bytes(hd)) / prefix_slot_bytes(hd, cache);
    return n < most ? n : most;
}
// Quantised rows wait in a ring of two tiles before they become fp16: bytes of a token's
// row there (off the banks of its neighbours'), and of a warp's tile: K rows, V rows, eight
// scales of each.
constexpr int prefix_raw_row(int hd, int cache) { return (cache == DTYPE_Q8_0 ? hd : hd / 2) + 16; }
constexpr int prefix_raw_tile(int hd, int cache) { return prefix_quant(cache) ? prefix_tile(hd, cache) / kConverters * 2 * (prefix_raw_row(hd, cache) + 32) : 0; }
constexpr size_t prefix_shared_bytes(int hd, int cache) {
    return 1024 + (size_t)prefix_streams(hd) * prefix_query_bytes(hd) + (size_t)prefix_slots(hd, cache) * prefix_slot_bytes(hd, cache) +
           2 * kConverters * prefix_raw_tile(hd, cache);
}
#ifdef __CUDACC__
// The prefix's tokens: its length, within its table.
__device__ __forceinline__ long long prefix_length(const PrefixParams &p, bool report) {
    long long n = __ldg(p.length);
    const long long room = min((long long)p.table_pages * p.l.page_size, kAttnMaxTokens);
    if (n < 0 || n > room) {
        if (report) atomicOr(p.err, kErrCache);
        n = n < 0 ? 0 : room;
    }
    return n;
}

// Two sums or products of fp32 in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
        " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n"
        " mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// The larger, or NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }      // e in -126 .. 127

// 16 bytes from global to shared memory, or zeros.
__device__ __forceinline__ void copy16_zfill(uint32_t dst, const uint8_t *src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
// Magnitudes, ordered like their bits, of those that are finite.
__device__ __forceinline__ uint32_t finite_bits(uint32_t x) {
    x &= 0x7fffffffu;
    return x < 0x7f800000u ? x : 0u;
}
// The power of two that a group's largest magnitude (its bits: of a value, or of a scale)
// is divided by, to go to [2^14, 2^15).
// (Of scales at most 2^96: 24 more has to be a power of two in fp32.)
template <int kCache>
__device__ __forceinline__ int prefix_exponent(uint32_t top) {
    top = __reduce_max_sync(0xffffffffu, top);
    return top == 0 ? -100 : min(max((int)(top >> 23) - 127 - 14, -100), prefix_quant(kCache) ? 96 : 113);
}

// Where an operand's row has dim d of each eight: Q4_0's codes stay as two words side by
// side give them (0 4 1 5 2 6 3 7), for queries and outputs are put in that order for less.
template <int kCache>
__host__ __device__ constexpr int prefix_place(int d) { return kCache == DTYPE_Q4_0 ? 2 * (d & 3) + (d >> 2) : d; }

// A warp's quantised rows of a tile, which wait in shared memory (K rows, V rows, their
// scales), as fp16 into the slots of K and V, zeros where a token does not count.  A lane
// takes one block of 32 codes a round, which lie in 8 words nb apart, and writes them as 64
// neighbouring bytes.
template <int kCache, int HD>
__device__ __forceinline__ void prefix_unpack(const uint8_t *raw, uint32_t valid, int first_row, int lane, float k_down, float v_down, uint8_t *k_to, uint8_t *v_to) {
    constexpr int TN = prefix_tile(HD, kCache), GT = TN / kConverters, NB = HD / 32, kRow = prefix_raw_row(HD, kCache);
    const float *const scales = reinterpret_cast<const float *>(raw + 2 * GT * kRow);
    // A code's bits are an fp16 subnormal, 2^-24 times it (a nibble four bits up: 2^-20),
    // so one product and sum, rounded once, with the scale and its offset make it a value
    // (2^-24, 2^-20 of it, which the group's power of two makes up for).
#pragma unroll 1
    for (int k = lane; k < 2 * GT * NB; k += 32) {
        // (Eight neighbouring lanes write 4 rows' 2 neighbouring blocks, which lie on all banks.)
        const int pair = NB % 2 ? 0 : (k >> 3) % (NB / 2), t2 = NB % 2 ? k / NB : (k >> 3) / (NB / 2) * 4 + ((k >> 1) & 3), b = NB % 2 ? k - t2 * NB : 2 * pair + (k & 1);
        const int t = t2 < GT ? t2 : t2 - GT, row = first_row + t;
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i] = kCache == DTYPE_Q8_0 ? reinterpret_cast<const uint32_t *>(raw + t2 * kRow)[i * NB + b] : reinterpret_cast<const uint16_t *>(raw + t2 * kRow)[i * NB + b];
        const __half f = __float2half_rn((valid >> t) & 1 ? scales[t2 * 8 + b] * (t2 < GT ? k_down : v_down) : 0.0f);
        const __half2 mul = __half2half2(f), add = __half2half2(__float2half_rn(__half2float(f) * -0x1p-17f));      // 128 2^-24 and 8 2^-20
        uint8_t *at = (t2 < GT ? k_to : v_to) + (b >> 1) * (TN * 128) + row * 128;
        const int chunk = ((b & 1) * 4) ^ (row & 7);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            uint32_t c[4];
            if constexpr (kCache == DTYPE_Q8_0) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    c[2 * i] = __byte_perm(w[2 * u + i], 0u, 0x4140);
                    c[2 * i + 1] = __byte_perm(w[2 * u + i], 0u, 0x4342);
                }
            } else {
                // Code by code of two words, as prefix_place has them.
                const uint32_t x = w[2 * u] + w[2 * u + 1] * 65536u, y = x >> 8;
                c[0] = (x * 16u) & 0x00f000f0u;
                c[1] = x & 0x00f000f0u;
                c[2] = (y * 16u) & 0x00f000f0u;
                c[3] = y & 0x00f000f0u;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = half2_bits(__hfma2(*reinterpret_cast<const __half2 *>(&c[i]), mul, add));
            *reinterpret_cast<uint4 *>(at + ((chunk ^ u) << 4)) = make_uint4(c[0], c[1], c[2], c[3]);
        }
    }
}

// The largest finite magnitude of a warp's F32 or BF16 rows.
template <int kCache, int HD, int GT>
__device__ __forceinline__ uint32_t prefix_largest(const uint8_t *from, unsigned row16, uint32_t valid, int lane) {
    constexpr int PR = kCache == DTYPE_F32 ? HD / 4 : HD / 8;
    uint32_t top = 0;
#pragma unroll 4
    for (int k = lane; k < (GT * PR + 31) / 32 * 32; k += 32) {
        const int t = k / PR, c = k - t * PR;
        const unsigned at = __shfl_sync(0xffffffffu, row16, t & 31) + c;
        if (!((valid >> (t & 31)) & 1) || t >= GT) continue;
        const uint4 x = __ldg(reinterpret_cast<const uint4 *>(from + ((unsigned long long)at << 4)));
        const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (kCache == DTYPE_F32) top = max(top, finite_bits(v[j]));
            else top = max(top, max(finite_bits(v[j] << 16), finite_bits(v[j] & 0xffff0000u)));
        }
    }
    return top;
}
// They as fp16 into a slot, zeros where a token does not count.
template <int kCache, int HD, int TN>
__device__ __forceinline__ void prefix_convert(const uint8_t *from, unsigned row16, uint32_t valid, int first_row, int lane, float down, uint8_t *to) {
    constexpr int GT = TN / kConverters, PR = HD / 8, kWords = kCache == DTYPE_F32 ? 2 : 1;       // of 16 bytes in 8 values
#pragma unroll 4
    for (int k = lane; k < (GT * PR + 31) / 32 * 32; k += 32) {
        const int t = k / PR, c = k - t * PR, row = first_row + t;
        const unsigned at = __shfl_sync(0xffffffffu, row16, t & 31) + c * kWords;
        if (t >= GT) continue;
        uint32_t y[4] = {0, 0, 0, 0};
        if ((valid >> t) & 1) {
            float f[8];
            if constexpr (kCache == DTYPE_F32) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 x = __ldg(reinterpret_cast<const float4 *>(from + ((unsigned long long)(at + i) << 4)));
                    f[4 * i] = x.x, f[4 * i + 1] = x.y, f[4 * i + 2] = x.z, f[4 * i + 3] = x.w;
                }
            } else {
                const uint4 x = __ldg(reinterpret_cast<const uint4 *>(from + ((unsigned long long)at << 4)));
                const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = half2_bits(__floats2half2_rn(f[2 * i] * down, f[2 * i + 1] * down));
        }
        *reinterpret_cast<uint4 *>(to + (c >> 3) * (TN * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
    }
}

// kUnarmed: for sapphire_test_tc_unarmed.
template <int kCache, int HD, bool kBf16, bool kUnarmed>
__global__ void __launch_bounds__((kPrefixCopy + prefix_copiers(kCache, kBf16)) * 32, 1) prefix_kernel(const PrefixParams p) {
    constexpr int TN = prefix_tile(HD, kCache), kGroups = prefix_copiers(kCache, kBf16), GT = TN / kGroups, kSlots = prefix_slots(HD, kCache), NB = HD / 32;
    constexpr int kQueryBytes = prefix_query_bytes(HD), kSlotBytes = prefix_slot_bytes(HD, kCache), kMaxStreams = prefix_streams(HD);
    constexpr int kRunTiles = kRunTokens / TN, kTileRing = 8;
    constexpr bool kRaw = prefix_raw(kCache, kBf16);              // rows are copied as they are
    constexpr bool kQuant = prefix_quant(kCache);
    constexpr float kBias = kBf16 ? 0.0f : 7.0f, kLag = 8.0f;
    // Columns: the tiles' O, then their S, then their P.
    constexpr int kSCol = kMaxStreams * HD, kPCol = kSCol + kMaxStreams * TN, kPStep = (TN / 2 + 15) / 16 * 16;
    static_assert(kPCol + kMaxStreams * kPStep <= 512 && kSlots >= 3 && HD % 32 == 0 && TN % 16 == 0 && GT % 2 == 0 && GT <= 32 &&
                  prefix_shared_bytes(HD, kCache) <= kPrefixShared + 4096, "");
    // fp32 += A B, both K-major for S; B's rows are the product's K for O
    constexpr uint32_t kFormat = (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(kPrefixRows >> 4) << 24);
    constexpr uint32_t kIdescS = kFormat | ((uint32_t)(TN >> 3) << 17), kIdescO = kFormat | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t landed[kRaw ? kSlots : 1], full[kSlots], empty[kSlots], q_full, s_full[2], s_free[2], p_ready[2], p_done[2], done[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int s_abort;
    __shared__ float qmul[2][2][kPrefixRows];                     // [item's parity][tile of rows]
    __shared__ uint32_t counts[kTileRing][kGroups];                     // tokens of a group that count
    __shared__ float k_up[kTileRing][kGroups];                          // a group's keys are the operand's times this
    __shared__ int v_up[kTileRing][kGroups];                            // and its values times 2 to this
    volatile int *const abort_flag = &s_abort;
    constexpr uint64_t kLimit = kUnarmed ? kTestWaitNs : kWaitNs;
    auto withheld = [&](int which, bool first) { return kUnarmed && first && p.unarmed == which && blockIdx.x == 0; };
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    // Barriers and tensor memory need nothing of an earlier kernel.
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < kSlots; ++s) {
            if (kRaw) mbar_init(landed + s, kGroups + kGroups * 32);      // a lane of each copying warp, and all lanes' copies
            mbar_init(full + s, kRaw ? 1 : kGroups);
            mbar_init(empty + s, p.streams);                      // of the issuing warps
        }
        mbar_init(&q_full, kGroups);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(s_free + i, 4);
            mbar_init(p_ready + i, 4);
            mbar_init(p_done + i, 1);
            mbar_init(done + i, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kPrefixMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    pdl_wait();
    const uint32_t length = (uint32_t)prefix_length(p, blockIdx.x == 0 && threadIdx.x == 0);
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < p.counts; i += gridDim.x * blockDim.x) p.count[i] = 0;
    const PrefixRanges r = prefix_ranges(p.items, length, TN, p.blocks);        // (TN: p.tile)
    PrefixPiece mine{0, 0, 0};
    if (blockIdx.x < r.blocks) mine = prefix_piece(r, blockIdx.x);
    const int item0 = __shfl_sync(0xffffffffu, (int)mine.item, 0), tile0 = __shfl_sync(0xffffffffu, (int)mine.tile, 0);
    const int units = __shfl_sync(0xffffffffu, (int)mine.units, 0), tiles = __shfl_sync(0xffffffffu, (int)r.tiles, 0);
    auto fail = [&]() {
        *abort_flag = 1;
        atomicOr(p.err, 2);
    };
    // Tiles of rows of an item.
    auto streams_of = [&](int item) { return min(p.streams, (p.rows - (item % p.row_sets) * p.streams * kPrefixRows + kPrefixRows - 1) / kPrefixRows); };

    const uint32_t tmem = tmem_slot;
    // (Arithmetic, not arrays: an index that the compiler does not know would put them
    // into local memory, whose cache is what shared memory leaves.)
    auto s_col = [&](int i) { return tmem + (uint32_t)(kSCol + i * TN); };
    auto p_col = [&](int i) { return tmem + (uint32_t)(kPCol + i * kPStep); };
    auto o_col = [&](int i) { return tmem + (uint32_t)(i * HD); };
    uint8_t *const slots = smem + kMaxStreams * kQueryBytes;

    if (warp < kPrefixMma) {
        if constexpr (kRaw) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        // ------------------------------------------------------- softmax --
        const int i = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = s_col(i) + lanes, p_at = p_col(i) + lanes, o_at = o_col(i) + lanes;
        float m = -INFINITY, l = 0.0f, qm = 0.0f;                 // of the run
        float m_item = -INFINITY, l_item = 0.0f;                  // of the item's runs before it
        int e_run = -1000, item = item0, tile = tile0, run = 0;
        uint32_t turn = 0;                                        // tiles of this tile of rows
        bool first_run = true;
        int now = i < kMaxStreams && units > 0 ? streams_of(item) : 0;
        for (int n = 0; n < units; ++n) {
            const bool last = n + 1 == units || tile + 1 == tiles;
            if (i < now) {
                if (!wait_warp(s_full + i, turn & 1, abort_flag, kLimit)) {
                    if (lane == 0) fail();
                    break;
                }
                tc_fence_after();
                const int ring = n & (kTileRing - 1);
                if (run == 0 && first_run) qm = qmul[(item - item0) & 1][i][row];
                uint32_t word[kGroups];
                float qg[kGroups];
                int eg[kGroups];
                bool whole = true;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    word[g] = counts[ring][g];
                    whole = whole && word[g] == 0xffffffffu >> (32 - GT);
                    qg[g] = kRaw ? qm : fmaxf(qm * k_up[ring][g], 1.2e-38f);
                    eg[g] = kRaw ? 0 : v_up[ring][g];
                }
                // The row's scores, -inf where a token does not count.
                float s[TN];
                uint32_t *const raw = reinterpret_cast<uint32_t *>(s);
#pragma unroll
                for (int c = 0; c < TN; c += 32) {
                    if (c + 32 <= TN) tmem_load<32>(s_at + c, raw + c);
                    else tmem_load<16>(s_at + c, raw + c);
                }
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free + i);
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        if (!((word[j / GT] >> (j % GT)) & 1)) s[j] = -INFINITY;
                }
                // (A NaN among them makes every one of the row's probabilities NaN.)
                float top = -INFINITY, top_value = -INFINITY;     // (the largest score; probability times value)
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    float t0 = s[g * GT], t1 = s[g * GT + 1];
#pragma unroll
                    for (int j = 2; j < GT; j += 2) {
                        t0 = max_nan(t0, s[g * GT + j]);
                        t1 = max_nan(t1, s[g * GT + j + 1]);
                    }
                    const float t2 = max_nan(t0, t1) * qg[g];
                    if (t2 != t2) qm = t2;
                    top = fmaxf(top, t2);
                    if (!kRaw) top_value = fmaxf(top_value, t2 + (float)eg[g]);
                }
                // ---- the tile before has left P and O ----
                if (turn > 0) {
                    if (!wait_warp(p_done + i, (turn - 1) & 1, abort_flag, kLimit)) {
                        if (lane == 0) fail();
                        break;
                    }
                    tc_fence_after();
                }
                // ---- the reference, and O in its units ----
                const bool grew = top > m + kLag || (m == -INFINITY && top > m) || (!kRaw && top_value - m > (float)e_run + kLag);
                if (__any_sync(0xffffffffu, grew)) {
                    const float mn = fmaxf(m, top);
                    float f = mn == -INFINITY ? 1.0f : attn_exp2(m - mn);
                    l *= f;
                    if (!kRaw) {
                        // (m + e_run never falls, so f is at most 1; -1000 is where there is no score.)
                        const int e = (int)ceilf(fmaxf(fmaxf(top_value - mn, (float)e_run + (m - mn)), -1000.0f));
                        if (mn != -INFINITY) f = attn_exp2((m - mn) + (float)(e_run - e));
                        e_run = e;
                    }
                    m = mn;
                    if (run > 0) {
#pragma unroll 1
                        for (int c = 0; c < HD; c += 16) {
                            float o[16];
                            tmem_load<16>(o_at + c, reinterpret_cast<uint32_t *>(o));
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] *= f;
                            tmem_store<16>(o_at + c, reinterpret_cast<uint32_t *>(o));
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : kBias - m;
                float2 sum[kGroups] = {};
#pragma unroll
                for (int c = 0; c < TN; c += 16) {
                    uint32_t w[8];
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const int j = c + k, g = j / GT;
                        const float mul = qm != qm ? qm : qg[g], at = kRaw ? ref : ref + (float)min(max(eg[g] - e_run, -100), 300);
                        const float2 x = fma2(make_float2(s[j], s[j + 1]), make_float2(mul, mul), make_float2(at, at));
                        const float2 y = make_float2(attn_exp2(x.x), attn_exp2(x.y));
                        sum[g] = add2(sum[g], y);
                        w[k / 2] = pack16<kBf16>(y.x, y.y);
                    }
                    tmem_store<8>(p_at + c / 2, w);
                }
#pragma unroll
                for (int g = 0; g < kGroups; ++g) l += kRaw ? sum[g].x + sum[g].y : (sum[g].x + sum[g].y) * pow2(min(max(e_run - eg[g], -126), 100));
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && !withheld(2, n == 0 && warp == 0)) mbar_arrive(p_ready + i);
                ++turn;
                if (++run == kRunTiles || last) {
                    // ---- the run's O, added to the item's ----
                    if (!wait_warp(p_done + i, (turn - 1) & 1, abort_flag, kLimit)) {
                        if (lane == 0) fail();
                        break;
                    }
                    tc_fence_after();
                    m -= kBias;
                    const size_t at = ((size_t)(blockIdx.x + item) * p.streams + i) * kPrefixRows + row;
                    float *to = p.part + at * HD;
                    const float top_ml = fmaxf(m, m_item), ref_ml = top_ml == -INFINITY ? 0.0f : top_ml;
                    const float w0 = l_item == 0.0f ? 0.0f : l_item * attn_exp2(m_item - ref_ml);
                    const float w1 = l == 0.0f ? 0.0f : l * attn_exp2(m - ref_ml), all = w0 + w1;
                    const float f0 = all == 0.0f ? 0.0f : w0 / all;
                    const float f1 = l == 0.0f ? 0.0f : (w1 / all) / l * (kRaw ? 1.0f : pow2(min(max(e_run, -126), 127)));
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
                        tmem_load<32>(o_at + c, reinterpret_cast<uint32_t *>(o));
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            float y[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                y[k] = l == 0.0f ? 0.0f : o[j + prefix_place<kCache>(k)] * f1;
                                if (!first_run) y[k] = fmaf(to[c + j + k], f0, y[k]);
                            }
                            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + c + j), "f"(y[0]), "f"(y[1]),
                                         "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7])
                                         : "memory");
                        }
                    }
                    tc_fence_before();
                    if (last) p.part_ml[at] = make_float2(top_ml, all);
                    // (The next item's rows know nothing of this one's.)
                    m_item = last ? -INFINITY : top_ml;
                    l_item = last ? 0.0f : all;
                    first_run = last;
                    m = -INFINITY;
                    l = 0.0f;
                    e_run = -1000;
                    run = 0;
                }
            }
            if (++tile == tiles) {
                tile = 0;
                ++item;
                if (n + 1 < units && i < kMaxStreams) now = streams_of(item);
            }
        }
    } else if (warp < kPrefixCopy) {
        if constexpr (kRaw) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        const int i = warp - kPrefixMma;                          // tile of rows
        if (i < p.streams) {
            // ------------------------------------------------------ MMAs --
            // A warp for each tile of rows, so that neither waits for the other's softmax.
            // The next tile's scores come before this one's outputs: the softmax has them
            // when it is done with this one.
            constexpr uint32_t kHigh = (1024u >> 4) | 1u << 14 | 2u << 29;  // stride, version, 128-byte swizzle
            const uint32_t q_low = ((saddr(smem) + i * kQueryBytes) >> 4) | 1u << 16, k_low = (saddr(slots) >> 4) | 1u << 16;
            const uint32_t v_low = (saddr(slots) >> 4) | (uint32_t)(TN * 128 >> 4) << 16;
            const uint32_t s_at = s_col(i), p_at = p_col(i), o_at = o_col(i);
            int item = item0, tile = tile0, run = 0, k_slot = 0, v_slot = 1;
            uint32_t k_phase = 0, v_phase = 0, q_phase = 0, s_turn = 0, p_turn = 0;
            auto step = [&](int &slot, uint32_t &phase) {         // two slots on
                slot += 2;
                if (slot >= kSlots) {
                    slot -= kSlots;
                    phase ^= 1;
                }
            };
            // (A tile of rows that an item does not have still gives its slots back.)
            auto scores = [&](bool active, bool new_item) {
                if (new_item && !wait_warp(&q_full, q_phase++ & 1, abort_flag, kLimit)) return false;
                if (!wait_warp(full + k_slot, k_phase, abort_flag, kLimit)) return false;
                if (active) {
                    if (s_turn > 0 && !wait_warp(s_free + i, (s_turn - 1) & 1, abort_flag, kLimit)) return false;
                    ++s_turn;
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j)
                        umma_ss(s_at, q_low + (j / 4) * (kPrefixRows * 128 >> 4) + (j % 4) * 2,
                                k_low + k_slot * (kSlotBytes >> 4) + (j / 4) * (TN * 128 >> 4) + (j % 4) * 2, kHigh, kIdescS, j > 0);
                    umma_commit_warp(s_full + i);
                    umma_commit_warp(empty + k_slot);
                } else if (lane == 0) {
                    mbar_arrive(empty + k_slot);
                }
                step(k_slot, k_phase);
                return true;
            };
            auto outputs = [&](bool active) {
                if (!wait_warp(full + v_slot, v_phase, abort_flag, kLimit)) return false;
                if (active) {
                    if (!wait_warp(p_ready + i, p_turn++ & 1, abort_flag, kLimit)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < TN / 16; ++j)
                        umma_ts(o_at, p_at + 8 * j, v_low + v_slot * (kSlotBytes >> 4) + j * (2048 >> 4), kHigh, kIdescO, run > 0 || j > 0);
                    umma_commit_warp(p_done + i);
                    umma_commit_warp(empty + v_slot);
                } else if (lane == 0) {
                    mbar_arrive(empty + v_slot);
                }
                step(v_slot, v_phase);
                return true;
            };
            bool now = i < streams_of(item), ok = units == 0 || scores(now, true);
            for (int n = 0; ok && n < units; ++n) {
                const bool ends = tile + 1 == tiles, more = n + 1 < units;
                const bool next = ends && more ? i < streams_of(item + 1) : now;
                // (An item's first scores wait for its queries, which wait for the last one's
                // scores, so outputs go first there.)
                if (more && !ends) ok = scores(next, false);
                ok = ok && outputs(now);
                if (more && ends) ok = ok && scores(next, true);
                run = run + 1 == kRunTiles || ends ? 0 : run + 1;
                now = next;
                if (ends) ++item;
                tile = ends ? 0 : tile + 1;
            }
            if (!ok && lane == 0) fail();
            __syncwarp();
            umma_commit_warp(done + i);
            (void)wait_warp(done + i, 0, nullptr, kLimit);
        } else if (kRaw && i == 2) {
            // What has landed is handed to the tensor cores' proxy by a warp that nobody
            // waits for (by the issuing one: 500 cycles of every tile).
            int s = 0;
            uint32_t phase = 0;
            for (int index = 0; index < 2 * units; ++index) {
                if (!wait_warp(landed + s, phase, abort_flag, kLimit)) {
                    if (lane == 0) fail();
                    break;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(full + s);
                if (++s == kSlots) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    } else {
        if constexpr (kRaw) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // ----------------------------------------------------- producers --
        const int w = warp - kPrefixCopy;                         // its tokens: GT w .. of a tile
        bool ok = true;
        // Token `lane` of a tile: its page (-1: none) and slot.
        auto fetch = [&](int t, int &entry, int &slot) {
            const uint32_t tok = (uint32_t)t * TN + w * GT + lane;         // (at most a tile behind the length)
            entry = -1;
            slot = 0;
            if (lane < GT && tok < length) {
                int pg = (int)(((unsigned long long)tok * p.page_mul) >> 32);
                slot = (int)tok - pg * p.l.page_size;
                if (slot < 0) {
                    --pg;
                    slot += p.l.page_size;
                }
                entry = __ldg(p.table + pg);
            }
        };
        // Copies of a lane (of rows as they are): 16-byte piece 32 j + lane of the warp's
        // rows, and where it goes in a slot.
        constexpr int PR = HD / 8, kCopies = kRaw ? (GT * PR + 31) / 32 : 1;
        uint32_t to[kCopies];
        if constexpr (kRaw) {
#pragma unroll
            for (int j = 0; j < kCopies; ++j) {
                const int k = 32 * j + lane, t = k / PR, c = k - t * PR, row = w * GT + t;
                to[j] = saddr(slots) + (c >> 3) * (TN * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
            }
        }
        // Where a tile's tokens are: of token `lane` its page's and its row's offset (in 16
        // bytes) and its slot; which of them count.
        struct Tokens {
            unsigned page16, row16;
            int slot;
            uint32_t valid;
        };
        auto resolve = [&](int t, int entry, int slot) {
            Tokens x;
            const bool wanted = lane < GT && (uint32_t)t * TN + w * GT + lane < length, found = (unsigned)entry < (unsigned)p.l.num_pages;
            x.page16 = (found ? (unsigned)entry : 0u) * (unsigned)(p.l.page_bytes >> 4);
            x.row16 = x.page16 + (unsigned)(slot * (p.l.row_bytes >> 4));
            x.slot = slot;
            x.valid = __ballot_sync(0xffffffffu, found && wanted);
            if (wanted && !found) atomicOr(p.err, kErrCache);
            return x;
        };
        auto head_of = [&](int item) { return p.l.pages + (unsigned long long)(item / p.row_sets) * p.l.chunk_bytes; };
        auto after = [&](int t) { return t + 1 == tiles ? 0 : t + 1; };
        int item = item0, tile = tile0, entry, slot, ring = 0, next_slot = 0;
        uint32_t next_phase = 1;
        if (units > 0) fetch(tile, entry, slot);
        // ---- quantised rows on their way, a tile ahead ----
        constexpr int kRawTile = prefix_raw_tile(HD, kCache), kRawRow = prefix_raw_row(HD, kCache);
        uint8_t *const raw = slots + kSlots * kSlotBytes + w * 2 * kRawTile;
        int ahead_item = item0, ahead_tile = tile0;
        const uint8_t *ahead_head = head_of(item0);
        auto bring = [&](int n) {
            if (n < units) {
                const Tokens x = resolve(ahead_tile, entry, slot);
                if (n + 1 < units) fetch(after(ahead_tile), entry, slot);
                if (lane == 0) counts[n % kTileRing][w] = x.valid;
                const uint32_t dst = saddr(raw) + (n & 1) * kRawTile;
                if ((x.valid >> lane) & 1) {
                    const uint8_t *from = ahead_head + p.l.ks_off + ((unsigned long long)x.page16 << 4) + x.slot * p.l.scale_stride * 4;
                    const uint32_t at = dst + 2 * GT * kRawRow + lane * 32;
#pragma unroll
                    for (int h = 0; h < 2; ++h, from += p.l.vs_off - p.l.ks_off) {
                        if constexpr (NB <= 2) copy_bytes<8>(at + h * GT * 32, from);
                        else copy_bytes<16>(at + h * GT * 32, from);
                        if constexpr (NB > 4) copy_bytes<16>(at + h * GT * 32 + 16, from + 16);
                    }
                }
                constexpr int kPieces = kRawRow / 16 - 1;
#pragma unroll
                for (int j = 0; j < (GT * kPieces + 31) / 32; ++j) {
                    const int k = 32 * j + lane, t = k / kPieces, c = k - t * kPieces;
                    const unsigned src = __shfl_sync(0xffffffffu, x.row16, t & 31) + c;
                    if (t < GT && (x.valid >> t) & 1) {
                        const uint8_t *from = ahead_head + ((unsigned long long)src << 4);
                        copy_bytes<16>(dst + t * kRawRow + c * 16, from);
                        copy_bytes<16>(dst + (GT + t) * kRawRow + c * 16, from + p.l.v_off);
                    }
                }
                if (++ahead_tile == tiles) {
                    ahead_tile = 0;
                    ahead_head = head_of(++ahead_item);
                }
            }
            copies_commit();
        };
        if constexpr (kQuant) bring(0);
        const uint8_t *head = head_of(item);
        auto next_slots = [&]() {
            if (++next_slot == kSlots) {
                next_slot = 0;
                next_phase ^= 1;
            }
        };
        for (int n = 0; ok && n < units; ++n) {
            if constexpr (kQuant) {
                bring(n + 1);
                copies_wait<1>();
                __syncwarp();
                const uint8_t *const these = raw + (n & 1) * kRawTile;
                const uint32_t valid = counts[ring][w];
                int e[2];                                         // powers of two of the group's keys and values
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t top = 0;
                    if ((valid >> lane) & 1) {
                        const uint32_t *at = reinterpret_cast<const uint32_t *>(these + 2 * GT * kRawRow) + (h * GT + lane) * 8;
#pragma unroll
                        for (int b = 0; b < NB; ++b) top = max(top, finite_bits(at[b]));
                    }
                    e[h] = prefix_exponent<kCache>(top);
                }
                if (lane == 0) {
                    constexpr int kUp = kCache == DTYPE_Q8_0 ? 24 : 20;
                    k_up[ring][w] = pow2(e[0] + kUp);
                    v_up[ring][w] = e[1] + kUp;
                }
                const int k_slot = next_slot;
                ok = wait_warp(empty + next_slot, next_phase, abort_flag, kLimit);
                next_slots();
                ok = ok && wait_warp(empty + next_slot, next_phase, abort_flag, kLimit);
                if (!ok) {
                    if (lane == 0) fail();
                    break;
                }
                prefix_unpack<kCache, HD>(these, valid, w * GT, lane, pow2(-e[0]), pow2(-e[1]), slots + k_slot * kSlotBytes, slots + next_slot * kSlotBytes);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    if (!withheld(3, n == 0 && w == 0)) mbar_arrive(full + k_slot);
                    mbar_arrive(full + next_slot);
                }
                next_slots();
            } else {
                const Tokens now = resolve(tile, entry, slot);
                if (n + 1 < units) fetch(after(tile), entry, slot);
                if (lane == 0) counts[ring][w] = now.valid;
                int e[2] = {0, 0};
                unsigned from[kCopies];
                if constexpr (kRaw) {
#pragma unroll
                    for (int j = 0; j < kCopies; ++j) {
                        const int k = 32 * j + lane, t = k / PR;
                        from[j] = __shfl_sync(0xffffffffu, now.row16, t & 31) + (k - t * PR);
                    }
                } else {
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        e[half] = prefix_exponent<kCache>(prefix_largest<kCache, HD, GT>(head + (half ? p.l.v_off : 0), now.row16, now.valid, lane));
                    if (lane == 0) {
                        k_up[ring][w] = pow2(e[0]);
                        v_up[ring][w] = e[1];
                    }
                }
                // ---- K, then V ----
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    if (!wait_warp(empty + next_slot, next_phase, abort_flag, kLimit)) {
                        if (lane == 0) fail();
                        ok = false;
                        break;
                    }
                    const uint32_t at = next_slot * kSlotBytes;
                    const uint8_t *const rows = head + (half ? p.l.v_off : 0);
                    if constexpr (kRaw) {
                        if (now.valid == 0xffffffffu >> (32 - GT)) {
#pragma unroll
                            for (int j = 0; j < kCopies; ++j)
                                if (32 * (j + 1) <= GT * PR || 32 * j + lane < GT * PR) copy_bytes<16>(to[j] + at, rows + ((unsigned long long)from[j] << 4));
                        } else {
#pragma unroll 1
                            for (int j = 0; j < kCopies; ++j) {
                                const int k = 32 * j + lane, t = k / PR, c = k - t * PR, row = w * GT + t;
                                const unsigned src = __shfl_sync(0xffffffffu, now.row16, t & 31) + c;
                                if (t < GT)
                                    copy16_zfill(saddr(slots) + at + (c >> 3) * (TN * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                                                 rows + ((unsigned long long)src << 4), (now.valid >> t) & 1);
                            }
                        }
                        // (They arrive when they land, whatever this warp does meanwhile.)
                        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(saddr(landed + next_slot)) : "memory");
                        if (lane == 0 && !withheld(3, n == 0 && half == 0 && w == 0)) mbar_arrive(landed + next_slot);
                    } else {
                        prefix_convert<kCache, HD, TN>(rows, now.row16, now.valid, w * GT, lane, pow2(half ? -e[1] : -e[0]), slots + at);
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0 && !withheld(3, n == 0 && half == 0 && w == 0)) mbar_arrive(full + next_slot);
                    }
                    next_slots();
                }
            }
            ring = (ring + 1) % kTileRing;
            if (ok && (n == 0 || tile == 0)) {
                // ---- the item's queries ----
                if (n > 0) {
                    const int index = 2 * n - 2;                  // the last scores of the item before
                    if (!wait_warp(empty + index % kSlots, (index / kSlots) & 1, abort_flag, kLimit)) {
                        if (lane == 0) fail();
                        break;
                    }
                }
                // Rows by 16-byte copies, or by values where they lie anywhere; then, where
                // they are converted or turned, each thread its row in place.
                constexpr int kRows = kPrefixRows / kGroups;
                const int row = w * kRows + min(lane, kRows - 1), streams = streams_of(item);
                for (int i = 0; i < streams; ++i) {
                    const int at = ((item % p.row_sets) * p.streams + i) * kPrefixRows + row;
                    const int seq = at < p.rows ? at / p.group : -1;
                    const long long from = seq * p.q_ss + (long long)(item / p.row_sets * p.group + at - seq * p.group) * p.q_hs;
                    const uint32_t rows_there = __ballot_sync(0xffffffffu, seq >= 0);
                    if (p.q_wide) {
                        const uint32_t from16 = (uint32_t)(from >> 3);        // (within 64 GB, checked on the host)
#pragma unroll 1
                        for (int j = 0; j < kRows * PR / 32; ++j) {
                            const int k = 32 * j + lane, t = k / PR, c = k - t * PR, q_row = w * kRows + t;
                            const bool there = (rows_there >> t) & 1;
                            const uint32_t at16 = __shfl_sync(0xffffffffu, from16, t), src = there ? at16 + c : 0u;
                            copy16_zfill(saddr(smem) + i * kQueryBytes + (c >> 3) * (kPrefixRows * 128) + q_row * 128 + (((c & 7) ^ (q_row & 7)) << 4),
                                         static_cast<const uint8_t *>(p.q) + ((unsigned long long)src << 4), there);
                        }
                    } else {
#pragma unroll 1
                        for (int c = 0; c < PR && lane < kRows; ++c) {
                            uint16_t v[8] = {};
                            if (seq >= 0) {
#pragma unroll
                                for (int e = 0; e < 8; ++e) v[e] = __ldg(static_cast<const uint16_t *>(p.q) + from + 8 * c + e);
                            }
                            memcpy(smem + i * kQueryBytes + (c >> 3) * (kPrefixRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4), v, sizeof v);
                        }
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
                const bool convert = !kBf16 && p.io == DTYPE_BF16;
                const uint32_t sign = p.scale < 0.0f ? 0x80008000u : 0u;
                for (int i = 0; i < streams && lane < kRows; ++i) {
                    float up = 1.0f, mul = fmaxf(fabsf(p.scale), 1.2e-38f);
                    auto piece = [&](int c) { return reinterpret_cast<uint4 *>(smem + i * kQueryBytes + (c >> 3) * (kPrefixRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)); };
                    if (convert) {
                        uint32_t top = 0;                         // magnitudes are ordered like their bits
#pragma unroll 4
                        for (int c = 0; c < PR; ++c) {
                            const uint4 x = *piece(c);
                            const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) top = max(top, max(v[j] & 0x7fffu, (v[j] >> 16) & 0x7fffu));
                        }
                        if (top > 0 && top < 0x7f80u) {
                            const int e = min(141 - (int)(top >> 7), 126);        // the largest goes to [2^14, 2^15)
                            up = pow2(e);
                            mul = fmaxf(mul * pow2(-e), 1.2e-38f);
                        }
                    }
                    if (convert || sign || kCache == DTYPE_Q4_0) {
#pragma unroll 4
                        for (int c = 0; c < PR; ++c) {
                            const uint4 x = *piece(c);
                            uint32_t v[4] = {x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign};
                            if (convert) {
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    v[j] = half2_bits(__floats2half2_rn(__uint_as_float(v[j] << 16) * up, __uint_as_float(v[j] & 0xffff0000u) * up));
                            }
                            if (kCache == DTYPE_Q4_0)             // (prefix_place)
                                *piece(c) = make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632), __byte_perm(v[1], v[3], 0x5410), __byte_perm(v[1], v[3], 0x7632));
                            else *piece(c) = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                    }
                    qmul[(item - item0) & 1][i][row] = mul;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0 && !withheld(1, n == 0 && w == 0)) mbar_arrive(&q_full);
            }
            if (++tile == tiles) {
                tile = 0;
                head = head_of(++item);
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kPrefixMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int kCache, int HD, bool kBf16, bool kUnarmed = false>
cudaError_t prefix_launch(const PrefixParams &p, cudaStream_t st) {
    if constexpr (HD == 128 && !kUnarmed)
        if (p.unarmed) return prefix_launch<kCache, HD, kBf16, true>(p, st);
    constexpr size_t kBytes = prefix_shared_bytes(HD, kCache);
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = attn_allow(prefix_kernel<kCache, HD, kBf16, kUnarmed>, kBytes, p.device, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(prefix_kernel<kCache, HD, kBf16, kUnarmed>, dim3(p.blocks), dim3((kPrefixCopy + prefix_copiers(kCache, kBf16)) * 32), kBytes, st, p);
}
template <int kCache, bool kBf16>
cudaError_t prefix_launch(const PrefixParams &p, cudaStream_t st) {
    switch (p.l.head_dim) {
        case 64: return prefix_launch<kCache, 64, kBf16>(p, st);
        case 96: return prefix_launch<kCache, 96, kBf16>(p, st);
        case 128: return prefix_launch<kCache, 128, kBf16>(p, st);
        case 192: return prefix_launch<kCache, 192, kBf16>(p, st);
        default: return prefix_launch<kCache, 256, kBf16>(p, st);
    }
}
#endif

// One cache type each (prefix_<type>.cu).
cudaError_t prefix_run_f32(const PrefixParams &p, cudaStream_t st);
cudaError_t prefix_run_bf16(const PrefixParams &p, cudaStream_t st);
cudaError_t prefix_run_f16(const PrefixParams &p, cudaStream_t st);
cudaError_t prefix_run_q8_0(const PrefixParams &p, cudaStream_t st);
cudaError_t prefix_run_q4_0(const PrefixParams &p, cudaStream_t st);
