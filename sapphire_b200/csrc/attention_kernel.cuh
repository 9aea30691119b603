// attention_kernel.cuh - one pass of attention of one new token over a paged
// cache; attention.cu plans and launches it.  Each cache type is compiled in a
// source of its own (attention_<type>.cu).
//
// Mathematics.  Per query head a running maximum m (of scores in units of
// log2 e), sum l and unnormalised acc = sum_t 2^(s_t - m + kBias) v_t; pieces
// of a sequence join by weights 2^(m_piece - m).
//
// What bounds it: every visible K and V row is read once from HBM, so the work
// is laid out to stream rows and to keep everything else off that path.
//
// Layout.  A warp takes 16 tokens at a time.  Scores are S^T = K Q^T and
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
// A tcgen05 tile would leave 120 of its 128 rows empty here; the MMAs below are
// a few percent of the pass.  K and V fragments go from global memory straight
// to registers as 16-byte loads: the order of dims inside an MMA is free as
// long as both operands share it, so a lane's consecutive bytes of a row are
// its fragment.
//
//   K (A operand): lane (g, t) = (lane / 4, lane % 4) loads rows g and g + 8,
//     dims 8t .. 8t + 7 of each 32.
//   V (A operand, transposed): lane (g, t) loads tokens 2t, 2t + 1, 2t + 8,
//     2t + 9, dims 8g .. 8g + 7 of each 64, and pairs tokens with byte permutes.
//   P (B operand): a movmatrix of the packed (high, low) pairs.
//
// Quantised rows are kept as words of 4 codes in the order [8][nb], so the same
// lanes read consecutive bytes; codes become fp16 exactly (1024 + code - 1152,
// or - 1032).  K's scale multiplies the 32-dim partial score; V's scale is
// multiplied into the probability (one B operand per 32 dims), brought into
// fp16's range by a power of two per warp that grows with the scales seen.
//
// Split.  The tiles (64 tokens of one KV head and up to 8 query heads) of all
// sequences are numbered in a row and cut into as many equal ranges as the GPU
// holds blocks, whatever the lengths; a block's pieces that do not hold a whole
// sequence go to the workspace and attend_join_kernel adds them up.
#pragma once

#include "attention.cuh"

constexpr int kAttnWarps = 4;
constexpr int kAttnTile = 16 * kAttnWarps;    // tokens of one tile
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
    KvLayout l;
    const void *q;
    void *out;
    float *lse;
    long long q_ss, q_hs, out_ss, out_hs;
    const int *page_table, *lengths;
    int io;                        // tensor_dtype_t of q and out
    int sequences, heads, group;   // group: query heads of a KV head
    int head_tiles;                // tiles of 4 NT query heads of a group
    int table_stride, length_offset, window;
    float scale;                   // scores times log2 e
    unsigned long long page_mul;   // floor(2^32 / page_size) + 1
    int blocks;
    float *part;                   // [blocks][2][GH * (HD + 2)]
    int4 *piece;                   // [blocks] (sequence, head tile, blocks it spans, -)
    int *err;
};

// Query heads of a tile for a group of this size.
inline bool attn_wide(int group) { return group > 4; }
inline int attn_tile_heads(int group) { return attn_wide(group) ? 8 : 4; }
// Resident blocks per SM that each variant is compiled for.
constexpr int attn_blocks_per_sm(int cache, int hd) {
    const bool quant = cache == DTYPE_Q8_0 || cache == DTYPE_Q4_0;
    return quant ? (hd <= 128 ? 4 : hd <= 192 ? 3 : 2) : (hd <= 96 ? 4 : hd <= 192 ? 3 : 2);
}

#ifdef __CUDACC__

// 2^(p + kBias): probabilities use the upper end of fp16 where the MMA is fp16.
template <int kCache>
constexpr float kAttnBias = (kCache == DTYPE_BF16 || kCache == DTYPE_F32) ? 0.0f : 14.0f;

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
// The 11 leading bits of x, rounded.
__device__ __forceinline__ uint32_t round_tf32(float x) {
    uint32_t y;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
    return y;
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
__device__ __forceinline__ float take_tf32(float &x) {
    const float hi = __uint_as_float(round_tf32(x));
    x -= hi;
    return hi;
}

// Two bytes of `w` (selected by sel's low nibbles of positions 0 and 2) as fp16
// integers - 128.
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t w, uint32_t sel) {
    const uint32_t x = __byte_perm(w, 0x64646464u, sel);          // 1024 + code
    const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&x), __half2half2(__ushort_as_half(0x6480)));   // - 1152
    return *reinterpret_cast<const uint32_t *>(&v);
}
// Nibbles 0 and 4 (kShift = 0), or 1 and 5 (kShift = 4), of w as fp16 integers - 8.
template <int kShift>
__device__ __forceinline__ uint32_t nibbles_to_half2(uint32_t w) {
    if (kShift == 0) {
        const uint32_t x = (w & 0x000f000fu) | 0x64006400u;       // 1024 + code
        const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&x), __half2half2(__ushort_as_half(0x6408)));
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const uint32_t x = (w & 0x00f000f0u) | 0x64006400u;           // 1024 + 16 code
    const __half2 v = __hfma2(*reinterpret_cast<const __half2 *>(&x), __half2half2(__ushort_as_half(0x2c00)),
                              __half2half2(__ushort_as_half(0xd480)));   // / 16 - 72
    return *reinterpret_cast<const uint32_t *>(&v);
}

// N bytes at p (aligned to the largest power of two up to 16 that divides N)
// into 32-bit words; zeros where !ok.
template <int N>
__device__ __forceinline__ void load_bytes(const uint8_t *p, bool ok, uint32_t *w) {
    if constexpr (N % 16 == 0) {
#pragma unroll
        for (int i = 0; i < N / 16; ++i) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (ok)
                asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                             : "l"(p + 16 * i));
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
    } else if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            uint2 u = make_uint2(0, 0);
            if (ok) u = __ldg(reinterpret_cast<const uint2 *>(p) + i);
            w[2 * i] = u.x, w[2 * i + 1] = u.y;
        }
    } else if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = ok ? __ldg(reinterpret_cast<const uint32_t *>(p) + i) : 0u;
    } else {
        static_assert(N % 2 == 0, "");
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const uint32_t h = ok ? __ldg(reinterpret_cast<const uint16_t *>(p) + i) : 0u;
            if (i % 2 == 0) w[i / 2] = h;
            else w[i / 2] |= h << 16;
        }
    }
}
template <int N>
__device__ __forceinline__ void load_scales(const uint8_t *p, bool ok, float (&s)[N]) {
    constexpr int kPad = N <= 2 ? 2 : N <= 4 ? 4 : 8;
    float f[kPad];
    load_bytes<kPad * 4>(p, ok, reinterpret_cast<uint32_t *>(f));
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = f[i];
}

// Shapes of one variant.
template <int kCache, int HD>
struct AttnShape {
    static constexpr bool kQuant = kCache == DTYPE_Q8_0 || kCache == DTYPE_Q4_0;
    static constexpr bool kF32 = kCache == DTYPE_F32;
    static constexpr bool kBf16 = kCache == DTYPE_BF16;
    static constexpr int NB = HD / 32;
    // Dims of one register chunk: 32 registers of K (or V) a lane.
    static constexpr int kChunk = kQuant ? HD : kF32 ? 64 : 128;
    static constexpr int kChunks = (HD + kChunk - 1) / kChunk;
    // Registers of a chunk: 2 K rows (4 lanes share a row) or 4 V rows (8 lanes).
    static constexpr int kRegs = kCache == DTYPE_Q8_0 ? HD / 8 : kCache == DTYPE_Q4_0 ? (HD / 16 < 8 ? 8 : HD / 16) : 32;
    static constexpr int kScaleBytes = NB <= 2 ? 8 : NB <= 4 ? 16 : 32;
    static constexpr int kChunkBytes = 256;                       // of a dense row
    static constexpr int kRowBytes = kCache == DTYPE_Q8_0 ? HD : kCache == DTYPE_Q4_0 ? HD / 2 : kF32 ? 4 * HD : 2 * HD;
    // Query parts in shared memory: rows of 8 columns, padded so that the rows
    // of neighbouring lanes fall on the other half of the banks.
    static constexpr int kQElem = kF32 ? 4 : 2;
    static constexpr int kQStride = (HD * kQElem) % 128 == 0 ? HD * kQElem + 64 : HD * kQElem;
};

// The positions a sequence's new token attends to, as tiles.
struct AttnSpan {
    int first, end, tile0, tiles;
};
__device__ __forceinline__ AttnSpan attn_span(const AttnParams &p, int s, bool report) {
    long long n = (long long)__ldg(p.lengths + s) + p.length_offset;
    const long long room = min((long long)p.table_stride * p.l.page_size, 0x7fffffc0ll);
    if (n < 0 || n > room) {
        if (report) atomicOr(p.err, kErrCache);
        n = n < 0 ? 0 : room;
    }
    AttnSpan a;
    a.end = (int)n;
    a.first = p.window > 0 && a.end > p.window ? a.end - p.window : 0;
    a.tile0 = a.first / kAttnTile;
    a.tiles = max(1, (a.end + kAttnTile - 1) / kAttnTile - a.tile0);      // an empty sequence still writes its zeros
    return a;
}

// kQS, kPS: B operands of a query and of a probability (narrow: one holds two
// parts, two hold three; wide: one part each).  kAligned: pages hold a multiple
// of 16 tokens, so a warp's tile lies in one page.
template <int kCache, int HD, bool kWide, int kQS, int kPS, bool kAligned>
__global__ void __launch_bounds__(kAttnWarps * 32, attn_blocks_per_sm(kCache, HD)) attend_kernel(const AttnParams p) {
    using Sh = AttnShape<kCache, HD>;
    constexpr int GH = kWide ? 8 : 4, HL = kWide ? 2 : 1;         // heads of a tile, and of a lane
    constexpr int NB = Sh::NB, kRegs = Sh::kRegs, kMTiles = HD / 16, C = Sh::kChunks;
    constexpr bool kBf16 = Sh::kBf16, kF32 = Sh::kF32;
    constexpr float kBias = kAttnBias<kCache>;
    // The query's parts; at the end of an item, the warps' outputs.
    constexpr int kQBytes = kQS * 8 * Sh::kQStride, kAccBytes = kAttnWarps * GH * HD * 4;
    __shared__ __align__(16) uint8_t sq[kQBytes > kAccBytes ? kQBytes : kAccBytes];
    float *const sacc = reinterpret_cast<float *>(sq);            // [warp][head][dim]
    __shared__ float sm_m[kAttnWarps][GH], sm_l[kAttnWarps][GH];
    __shared__ float qmul[GH];
    __shared__ long long warp_sum[kAttnWarps];
    __shared__ int found_seq;
    __shared__ long long found_base;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_trigger();

    // ---- this block's range of tiles [lo, hi) of all sequences' ----
    const int per_thread = (p.sequences + kAttnWarps * 32 - 1) / (kAttnWarps * 32);
    const int s0 = min(tid * per_thread, p.sequences), s1 = min(s0 + per_thread, p.sequences);
    const int rows = p.l.kv_heads * p.head_tiles;                 // items of a sequence
    long long mine = 0;
    for (int s = s0; s < s1; ++s) mine += attn_span(p, s, blockIdx.x == 0).tiles;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    long long total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
        if (w < warp) before += warp_sum[w];
        total += warp_sum[w];
    }
    long long base = (before + incl - mine) * rows;
    total *= rows;
    const int blocks = (int)min((long long)p.blocks, total);
    const int bid = blockIdx.x;
    if (bid >= blocks) {
        if (tid == 0) p.piece[bid] = make_int4(0, 0, 0, 0);
        return;
    }
    const long long lo = bid * total / blocks, hi = (bid + 1) * total / blocks;
    if (lo >= base && lo < base + mine * rows) {
        for (int s = s0; s < s1; ++s) {
            const long long n = (long long)attn_span(p, s, false).tiles * rows;
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
    long long seq_base = found_base;
    int4 piece = make_int4(0, 0, 0, 0);

    long long pos = lo;
    while (pos < hi) {
        AttnSpan sp = attn_span(p, seq, false);
        if (pos >= seq_base + (long long)sp.tiles * rows) {
            seq_base += (long long)sp.tiles * rows;
            ++seq;
            continue;
        }
        const int item = (int)((pos - seq_base) / sp.tiles);      // (KV head, head tile)
        const long long item0 = seq_base + (long long)item * sp.tiles;
        const long long end = min(hi, item0 + sp.tiles);
        const int kh = item / p.head_tiles, ht = item - kh * p.head_tiles;
        const int nh = min(GH, p.group - ht * GH);                // heads of this tile
        const int head0 = kh * p.group + ht * GH;
        const uint8_t *head = p.l.pages + (unsigned long long)kh * p.l.chunk_bytes;
        const int *table = p.page_table + (long long)seq * p.table_stride;
        const unsigned page16 = (unsigned)(p.l.page_bytes >> 4);
        const int tile_first = sp.tile0 + (int)(pos - item0), tile_end = sp.tile0 + (int)(end - item0);

        // ---- where a tile's tokens are ----
        // A tile's page ids are fetched a tile ahead (fetch) and then resolved
        // to the 16-byte offset of the page, the slot and the tokens that
        // count.  Lane l looks up token l % 16; pages of a multiple of 16
        // tokens need one look-up, which every lane makes alike.
        int entry, slot, tok0;
        auto fetch = [&](int tile) {
            tok0 = tile * kAttnTile + warp * 16;
            const int tok = kAligned ? tok0 : tok0 + (lane & 15);
            int pg = (int)(((unsigned long long)(unsigned)tok * p.page_mul) >> 32);
            slot = tok - pg * p.l.page_size;
            if (slot < 0) {
                --pg;
                slot += p.l.page_size;
            }
            const bool inside = kAligned ? tok0 + 16 > sp.first && tok0 < sp.end : tok >= sp.first && tok < sp.end;
            entry = inside ? __ldg(table + pg) : -1;
        };
        unsigned at16 = 0, valid = 0;
        int at_slot = 0;
        const uint8_t *at_page = head;
        auto resolve = [&]() {
            const bool ok = (unsigned)entry < (unsigned)p.l.num_pages;
            const int l0 = max(sp.first - tok0, 0), l1 = min(sp.end - tok0, 16);
            unsigned inside = l1 > l0 ? (0xffffu >> (16 - l1)) & (0xffffu << l0) : 0u;
            at_slot = slot;
            if constexpr (kAligned) {
                if (inside && !ok) {
                    if (lane == 0) atomicOr(p.err, kErrCache);
                    inside = 0;
                }
                valid = inside;
                at_page = head + (ok ? (unsigned long long)((unsigned)entry * page16) << 4 : 0ull);
            } else {
                valid = __ballot_sync(0xffffffffu, ok) & inside;
                if (lane < 16 && ((inside >> lane) & 1) && !ok) atomicOr(p.err, kErrCache);
                at16 = ok ? (unsigned)entry * page16 : 0u;
            }
        };
        auto row_ptr = [&](int token, int off, int stride) {
            if constexpr (kAligned) return at_page + (off + (at_slot + token) * stride);
            const unsigned o16 = __shfl_sync(0xffffffffu, at16, token);
            const int sl = __shfl_sync(0xffffffffu, at_slot, token);
            return head + ((unsigned long long)o16 << 4) + (unsigned)(off + sl * stride);
        };

        // ---- rows to registers: chunk c of K (c < C) and of V (c - C) ----
        uint32_t buf[2][kRegs];
        float ks[2][NB], vs[2][NB];
        auto load = [&](int i) {
            uint32_t *w = buf[i & 1];
            if (i < C) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const bool ok = (valid >> (g + 8 * r)) & 1;
                    const uint8_t *row = row_ptr(g + 8 * r, 0, Sh::kRowBytes);
                    if constexpr (Sh::kQuant) {
                        constexpr int kBytes = Sh::kRowBytes / 4;
                        load_bytes<kBytes>(row + t * kBytes, ok, w + r * (kBytes / 4));
                        load_scales<NB>(row_ptr(g + 8 * r, p.l.ks_off, Sh::kScaleBytes), ok, ks[r]);
                    } else {
                        // 64 bytes of the row at a time, 16 of them this lane's
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (i * Sh::kChunkBytes + 64 * j < Sh::kRowBytes)
                                load_bytes<16>(row + i * Sh::kChunkBytes + 64 * j + 16 * t, ok, w + r * 16 + 4 * j);
                    }
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int tok = kF32 ? t + 4 * r : 2 * t + (r & 1) + 8 * (r >> 1);
                    const bool ok = (valid >> tok) & 1;
                    const uint8_t *row = row_ptr(tok, p.l.v_off, Sh::kRowBytes);
                    if constexpr (Sh::kQuant) {
                        constexpr int kBytes = Sh::kRowBytes / 8;
                        load_bytes<kBytes>(row + g * kBytes, ok, w + r * ((kBytes + 3) / 4));
                    } else {
                        // 128 bytes of the row at a time (64 where the head ends), 16 (8) of them this lane's
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int off = (i - C) * Sh::kChunkBytes + 128 * j;
                            if (off + 128 <= Sh::kRowBytes) load_bytes<16>(row + off + 16 * g, ok, w + r * 8 + 4 * j);
                            else if (off + 64 <= Sh::kRowBytes) load_bytes<8>(row + off + 8 * g, ok, w + r * 8 + 4 * j);
                        }
                    }
                }
                if constexpr (Sh::kQuant) {
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        load_scales<NB>(row_ptr(g + 8 * r, p.l.vs_off, Sh::kScaleBytes), (valid >> (g + 8 * r)) & 1, vs[r]);
                }
            }
        };
        // After chunk i is used, its registers take chunk i + 2, of the next
        // tile where this one has no more.
        auto load_after = [&](int i, int tile) {
            if (i + 2 < 2 * C) {
                load(i + 2);
            } else if (tile + 1 < tile_end) {
                if (i == 2 * C - 2) {
                    resolve();
                    load(0);
                    if (tile + 2 < tile_end) fetch(tile + 2);
                } else {
                    load(1);
                }
            }
        };

        // ---- the first tile's rows on their way, then the query's parts in
        //      shared memory in B operand order ----
        fetch(tile_first);
        constexpr int kPerWarp = GH / kAttnWarps;
        float x[kPerWarp][NB];
#pragma unroll
        for (int k = 0; k < kPerWarp; ++k) {
            const int j = warp + k * kAttnWarps;
            const long long off = seq * p.q_ss + (long long)(head0 + j) * p.q_hs + lane;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                x[k][b] = j >= nh ? 0.0f
                          : p.io == DTYPE_F32  ? __ldg(static_cast<const float *>(p.q) + off + 32 * b)
                          : p.io == DTYPE_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p.q)[off + 32 * b])
                                               : __half2float(static_cast<const __half *>(p.q)[off + 32 * b]);
        }
        resolve();
        load(0);
        load(1);
        if (tile_first + 1 < tile_end) fetch(tile_first + 1);
        __syncthreads();                                          // the last item's readers
#pragma unroll
        for (int k = 0; k < kPerWarp; ++k) {
            const int j = warp + k * kAttnWarps;
            float up = 1.0f, mul = p.scale;
            if (!kBf16 && !kF32) {
                // fp16 parts: the head's largest value goes to [2^14, 2^15).
                float top = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b) top = fmaxf(top, fabsf(x[k][b]));
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                if (top > 0.0f && top < INFINITY) {
                    const int e = min(max(14 - ilogbf(top), -126), 126);
                    up = ldexpf(1.0f, e);
                    mul = p.scale * ldexpf(1.0f, -e);
                }
            }
            if (lane == 0) qmul[j] = mul;
            const int col = kWide ? j : 2 * j;
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
        float qm[HL];
#pragma unroll
        for (int j = 0; j < HL; ++j) qm[j] = qmul[HL * t + j];

        // ---- the pass over this block's tiles of the item ----
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
        float vlim = 0.0f, vinv = 0.0f;                           // V scales: largest that fits, and the power of two
        for (int tile = tile_first; tile < tile_end; ++tile) {
            const bool ok0 = (valid >> g) & 1, ok1 = (valid >> (g + 8)) & 1;
            // ---- scores of 16 tokens: lane (g, t) has tokens g, g + 8 of its heads ----
            float s[HL][2];
            if constexpr (Sh::kQuant) {
                const uint32_t *kr = buf[0];
#pragma unroll
                for (int j = 0; j < HL; ++j) s[j][0] = s[j][1] = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t a[2][4];
                    constexpr int kW = Sh::kRowBytes / 16;            // words of a row in this lane
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        if constexpr (kCache == DTYPE_Q8_0) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint32_t w = kr[r * kW + i * NB + b];
                                a[i][r] = bytes_to_half2(w, 0x4140);
                                a[i][2 + r] = bytes_to_half2(w, 0x4342);
                            }
                        } else {
                            // halfwords b and NB + b: codes 0-3 of words 2t and 2t + 1
                            const uint32_t u = kr[r * kW + b / 2], v = kr[r * kW + (NB + b) / 2];
                            const uint32_t w = __byte_perm(u, v, (b & 1 ? 0x32 : 0x10) | ((NB + b) & 1 ? 0x7600 : 0x5400));
                            a[0][r] = nibbles_to_half2<0>(w);
                            a[0][2 + r] = nibbles_to_half2<4>(w);
                            a[1][r] = nibbles_to_half2<0>(w >> 8);
                            a[1][2 + r] = nibbles_to_half2<4>(w >> 8);
                        }
                    }
                    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int set = 0; set < kQS; ++set) {
                        const uint4 q = *reinterpret_cast<const uint4 *>(sq + (set * 8 + g) * Sh::kQStride + 64 * b + 16 * t);
                        mma16<false>(c, a[0][0], a[0][1], a[0][2], a[0][3], q.x, q.y);
                        mma16<false>(c, a[1][0], a[1][1], a[1][2], a[1][3], q.z, q.w);
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        if constexpr (kWide) {
                            s[0][r] = fmaf(ks[r][b], c[2 * r], s[0][r]);
                            s[1][r] = fmaf(ks[r][b], c[2 * r + 1], s[1][r]);
                        } else {
                            s[0][r] = fmaf(ks[r][b], c[2 * r] + c[2 * r + 1], s[0][r]);
                        }
                    }
                }
                load_after(0, tile);
            } else {
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ch = 0; ch < C; ++ch) {
                    const uint32_t *kr = buf[ch & 1];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int off = ch * Sh::kChunkBytes + 64 * i;            // bytes into the row
                        if (off >= Sh::kRowBytes) continue;
                        const uint32_t *u = kr + 4 * i, *v = kr + 16 + 4 * i;
                        uint32_t uh[4], ul[4], vh[4], vl[4];
                        if constexpr (kF32) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                float a = __uint_as_float(u[j]), b = __uint_as_float(v[j]);
                                uh[j] = __float_as_uint(take_tf32(a));
                                vh[j] = __float_as_uint(take_tf32(b));
                                ul[j] = round_tf32(a);
                                vl[j] = round_tf32(b);
                            }
                        }
#pragma unroll
                        for (int set = 0; set < kQS; ++set) {
                            const uint4 q = *reinterpret_cast<const uint4 *>(sq + (set * 8 + g) * Sh::kQStride + off + 16 * t);
                            if constexpr (kF32) {
                                mma_tf32(c, ul[0], vl[0], ul[1], vl[1], q.x, q.y);
                                mma_tf32(c, ul[2], vl[2], ul[3], vl[3], q.z, q.w);
                                mma_tf32(c, uh[0], vh[0], uh[1], vh[1], q.x, q.y);
                                mma_tf32(c, uh[2], vh[2], uh[3], vh[3], q.z, q.w);
                            } else {
                                mma16<kBf16>(c, u[0], v[0], u[1], v[1], q.x, q.y);
                                mma16<kBf16>(c, u[2], v[2], u[3], v[3], q.z, q.w);
                            }
                        }
                    }
                    load_after(ch, tile);
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if constexpr (kWide) {
                        s[0][r] = c[2 * r];
                        s[1][r] = c[2 * r + 1];
                    } else {
                        s[0][r] = c[2 * r] + c[2 * r + 1];
                    }
                }
            }
            // ---- probabilities ----
            float pr[HL][2], top[HL];
            bool grew = false;
#pragma unroll
            for (int j = 0; j < HL; ++j) {
                s[j][0] = ok0 ? s[j][0] * qm[j] : -INFINITY;
                s[j][1] = ok1 ? s[j][1] * qm[j] : -INFINITY;
                top[j] = fmaxf(s[j][0], s[j][1]);
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
                const float ref = m[j] == -INFINITY ? 0.0f : m[j] - kBias;
                pr[j][0] = attn_exp2(s[j][0] - ref);
                pr[j][1] = attn_exp2(s[j][1] - ref);
                l[j] += pr[j][0] + pr[j][1];
            }
            // The 16-bit B operands of w (tokens g and g + 8 of the lane's heads).
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
                            u = pack16<kBf16>(y[0], y[1]);
                            if (set + 1 < kPS) {
                                take16<kBf16>(y[0]);
                                take16<kBf16>(y[1]);
                            }
                        } else {
                            const float hi2 = take16<kBf16>(y[0]);
                            u = pack16<kBf16>(hi2, y[0]);
                            if (set + 1 < kPS) take16<kBf16>(y[0]);
                            if (set == 1) u = pack16<kBf16>(hi2, 0.0f);
                        }
                        (r ? b1 : b0)[set] = transpose8x8(u);
                    }
                }
            };
            // ---- acc += V^T P^T ----
            if constexpr (Sh::kQuant) {
                const uint32_t *vr = buf[1];
                float big = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b) big = fmaxf(big, fmaxf(fabsf(vs[0][b]), fabsf(vs[1][b])));
                if (__any_sync(0xffffffffu, big > vlim)) {
                    // A larger scale than fits: a new power of two that brings it to [1/2, 1).
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                    const int e = min(max((int)((__float_as_uint(big) >> 23) & 255) - 126, -126), 126);
                    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
                    const float f = vinv == 0.0f ? 0.0f : inv / vinv;
                    vinv = inv;
                    vlim = 3.5f / inv;
#pragma unroll
                    for (int i = 0; i < kMTiles; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][j] *= f;
                }
                constexpr int kW = (Sh::kRowBytes / 8 + 3) / 4;       // words of a row in this lane
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t a[2][4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        if constexpr (kCache == DTYPE_Q8_0) {
                            const uint32_t u = vr[(2 * r) * kW + b], v = vr[(2 * r + 1) * kW + b];
                            const uint32_t lo2 = __byte_perm(u, v, 0x5140), hi2 = __byte_perm(u, v, 0x7362);
                            a[0][2 * r] = bytes_to_half2(lo2, 0x4140);
                            a[0][2 * r + 1] = bytes_to_half2(lo2, 0x4342);
                            a[1][2 * r] = bytes_to_half2(hi2, 0x4140);
                            a[1][2 * r + 1] = bytes_to_half2(hi2, 0x4342);
                        } else {
                            const uint32_t w = __byte_perm(vr[(2 * r) * kW + b / 2], vr[(2 * r + 1) * kW + b / 2],
                                                           b & 1 ? 0x7632 : 0x5410);
                            a[0][2 * r] = nibbles_to_half2<0>(w);
                            a[0][2 * r + 1] = nibbles_to_half2<4>(w);
                            a[1][2 * r] = nibbles_to_half2<0>(w >> 8);
                            a[1][2 * r + 1] = nibbles_to_half2<4>(w >> 8);
                        }
                    }
                    const float f0 = vs[0][b] * vinv, f1 = vs[1][b] * vinv;
                    float w[HL][2];
#pragma unroll
                    for (int j = 0; j < HL; ++j) {
                        w[j][0] = pr[j][0] * f0;
                        w[j][1] = pr[j][1] * f1;
                    }
                    uint32_t b0[kPS], b1[kPS];
                    operand(w, b0, b1);
#pragma unroll
                    for (int set = 0; set < kPS; ++set) {
                        mma16<false>(acc[2 * b], a[0][0], a[0][1], a[0][2], a[0][3], b0[set], b1[set]);
                        mma16<false>(acc[2 * b + 1], a[1][0], a[1][1], a[1][2], a[1][3], b0[set], b1[set]);
                    }
                }
                load_after(1, tile);
            } else if constexpr (kF32) {
                // 32-bit B operands: column g is head g's part (wide), or part g % 2 of head g / 2.
                uint32_t pb[kPS][2][2];                               // [set][8 tokens][k = t, t + 4]
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float y[HL];
#pragma unroll
                    for (int j = 0; j < HL; ++j) y[j] = pr[j][r];
#pragma unroll
                    for (int set = 0; set < kPS; ++set) {
                        const float u = take_tf32(y[0]);
                        const float v = kWide ? take_tf32(y[HL - 1]) : __uint_as_float(round_tf32(y[0]));
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int src = (t + 4 * k) * 4 + (g >> 1);
                            const float a = __shfl_sync(0xffffffffu, u, src), b = __shfl_sync(0xffffffffu, v, src);
                            pb[set][r][k] = __float_as_uint(g & 1 ? b : a);
                        }
                    }
                }
#pragma unroll
                for (int ch = 0; ch < C; ++ch) {
                    const uint32_t *vr = buf[(C + ch) & 1];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {                     // 32 dims
                        const int d32 = ch * 2 + i;
                        if (d32 >= NB) continue;
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {             // tokens 8r .. 8r + 7
                                uint32_t h[4], lw[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    float y = __uint_as_float(vr[(2 * r + (k >> 1)) * 8 + 4 * i + 2 * j + (k & 1)]);
                                    h[k] = __float_as_uint(take_tf32(y));
                                    lw[k] = round_tf32(y);
                                }
#pragma unroll
                                for (int set = 0; set < kPS; ++set) {
                                    mma_tf32(acc[2 * d32 + j], lw[0], lw[1], lw[2], lw[3], pb[set][r][0], pb[set][r][1]);
                                    mma_tf32(acc[2 * d32 + j], h[0], h[1], h[2], h[3], pb[set][r][0], pb[set][r][1]);
                                }
                            }
                    }
                    load_after(C + ch, tile);
                }
            } else {
                uint32_t b0[kPS], b1[kPS];
                operand(pr, b0, b1);
#pragma unroll
                for (int ch = 0; ch < C; ++ch) {
                    const uint32_t *vr = buf[(C + ch) & 1];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int off = ch * Sh::kChunkBytes + 128 * i;           // bytes into the row
                        if (off >= Sh::kRowBytes) continue;
                        const int pairs = off + 128 <= Sh::kRowBytes ? 4 : 2;     // dims 2j, 2j + 1 of this lane
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (j >= pairs) continue;
                            const uint32_t x0 = vr[0 * 8 + 4 * i + j], x1 = vr[1 * 8 + 4 * i + j];
                            const uint32_t y0 = vr[2 * 8 + 4 * i + j], y1 = vr[3 * 8 + 4 * i + j];
                            const uint32_t a0 = __byte_perm(x0, x1, 0x5410), a1 = __byte_perm(x0, x1, 0x7632);
                            const uint32_t a2 = __byte_perm(y0, y1, 0x5410), a3 = __byte_perm(y0, y1, 0x7632);
#pragma unroll
                            for (int set = 0; set < kPS; ++set)
                                mma16<kBf16>(acc[off / 32 + j], a0, a1, a2, a3, b0[set], b1[set]);
                        }
                    }
                    load_after(C + ch, tile);
                }
            }
        }

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
        const bool whole = pos == item0 && end == item0 + sp.tiles;
        float *part = p.part + (size_t)(2 * bid + (pos == item0 ? 1 : 0)) * GH * (HD + 2);
        if (warp == 0 && g == 0) {
#pragma unroll
            for (int j = 0; j < HL; ++j) {
                const int h = HL * t + j;
                if (!whole) {
                    part[h] = M[j];
                    part[GH + h] = L[j];
                } else {
                    qmul[h] = L[j] == 0.0f ? 0.0f : 1.0f / L[j];
                    if (p.lse && h < nh)
                        p.lse[(long long)seq * p.heads + head0 + h] =
                            L[j] == 0.0f ? -INFINITY : (M[j] - kBias + log2f(L[j])) * 0.6931471805599453f;
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
                o *= qmul[h];
                const long long off = seq * p.out_ss + (long long)(head0 + h) * p.out_hs + d;
                if (p.io == DTYPE_F32) static_cast<float *>(p.out)[off] = o;
                else if (p.io == DTYPE_BF16) static_cast<__nv_bfloat16 *>(p.out)[off] = __float2bfloat16_rn(o);
                else static_cast<__half *>(p.out)[off] = __float2half_rn(o);
            }
        }
        if (pos == item0 && !whole) {
            // The blocks of this item: this one and all up to the one that holds its last tile.
            const long long last = ((item0 + sp.tiles) * blocks - 1) / total;
            piece = make_int4(seq, item, (int)(last - bid) + 1, 0);
        }
        pos = end;
    }
    if (tid == 0) p.piece[bid] = piece;
}

// Adds up an item that several blocks hold, one block per first holder, one
// warp per query head.
template <int HD, int GH>
__global__ void __launch_bounds__(GH * 32) attend_join_kernel(const AttnParams p, float bias) {
    pdl_wait();
    const int4 piece = __ldcg(p.piece + blockIdx.x);
    if (piece.z == 0) return;
    const int h = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kh = piece.y / p.head_tiles, ht = piece.y - kh * p.head_tiles;
    if (h >= min(GH, p.group - ht * GH)) return;
    constexpr int kStride = GH * (HD + 2), kVals = HD / 32;
    // Holder i's partial: the second slot of the first block, the first of the others.
    const float *part = p.part + (size_t)(2 * blockIdx.x + 1) * kStride;
    float M = -INFINITY;
    for (int i = lane; i < piece.z; i += 32) M = fmaxf(M, __ldcg(part + (size_t)(i ? 2 * i - 1 : 0) * kStride + h));
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float L = 0.0f, o[kVals];
#pragma unroll
    for (int j = 0; j < kVals; ++j) o[j] = 0.0f;
#pragma unroll 4
    for (int i = 0; i < piece.z; ++i) {
        const float *x = part + (size_t)(i ? 2 * i - 1 : 0) * kStride;
        const float w = M == -INFINITY ? 1.0f : attn_exp2(__ldcg(x + h) - M);
        L = fmaf(w, __ldcg(x + GH + h), L);
#pragma unroll
        for (int j = 0; j < kVals; ++j) o[j] = fmaf(w, __ldcg(x + 2 * GH + h * HD + 32 * j + lane), o[j]);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int head = kh * p.group + ht * GH + h;
    if (p.lse && lane == 0)
        p.lse[(long long)piece.x * p.heads + head] = L == 0.0f ? -INFINITY : (M - bias + log2f(L)) * 0.6931471805599453f;
    const long long off = piece.x * p.out_ss + (long long)head * p.out_hs + lane;
#pragma unroll
    for (int j = 0; j < kVals; ++j) {
        const float y = o[j] * inv;
        if (p.io == DTYPE_F32) static_cast<float *>(p.out)[off + 32 * j] = y;
        else if (p.io == DTYPE_BF16) static_cast<__nv_bfloat16 *>(p.out)[off + 32 * j] = __float2bfloat16_rn(y);
        else static_cast<__half *>(p.out)[off + 32 * j] = __float2half_rn(y);
    }
}

// The variant of a cache type for a head size: narrow or wide by the group,
// pages of a multiple of 16 tokens or any.
template <int kCache, int HD, bool kWide, int kQS, int kPS>
cudaError_t attn_launch(const AttnParams &p, cudaStream_t st) {
    if (p.l.page_size % 16 == 0)
        attend_kernel<kCache, HD, kWide, kQS, kPS, true><<<p.blocks, kAttnWarps * 32, 0, st>>>(p);
    else
        attend_kernel<kCache, HD, kWide, kQS, kPS, false><<<p.blocks, kAttnWarps * 32, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    constexpr int GH = kWide ? 8 : 4;
    return launch_pdl(attend_join_kernel<HD, GH>, dim3(p.blocks), dim3(GH * 32), 0, st, p, kAttnBias<kCache>);
}
template <int kCache, bool kWide, int kQS, int kPS>
cudaError_t attn_launch(const AttnParams &p, cudaStream_t st) {
    switch (p.l.head_dim) {
        case 64: return attn_launch<kCache, 64, kWide, kQS, kPS>(p, st);
        case 96: return attn_launch<kCache, 96, kWide, kQS, kPS>(p, st);
        case 128: return attn_launch<kCache, 128, kWide, kQS, kPS>(p, st);
        case 192: return attn_launch<kCache, 192, kWide, kQS, kPS>(p, st);
        default: return attn_launch<kCache, 256, kWide, kQS, kPS>(p, st);
    }
}
#endif

// One cache type each (attention_<type>.cu).  A bf16 query and output need
// fewer parts than the others where noted there.
cudaError_t attn_run_f32(const AttnParams &p, cudaStream_t st);
cudaError_t attn_run_bf16(const AttnParams &p, cudaStream_t st);
cudaError_t attn_run_f16(const AttnParams &p, cudaStream_t st);
cudaError_t attn_run_q8_0(const AttnParams &p, cudaStream_t st);
cudaError_t attn_run_q4_0(const AttnParams &p, cudaStream_t st);
