// prefix_kernel.cuh - attention of a whole batch's new tokens to a prefix that all
// of its sequences share, on the tensor cores (tcgen05); attention_shared.cu plans
// and launches it.  Each cache type is compiled in a source of its own.
//
// Mathematics.  The rows of a KV head are the query heads it serves, of every
// sequence: S = Q K^T over the prefix, P = 2^(S - m), O = P V, with a running
// maximum m and sum l a row.  A piece of the prefix leaves O / l, m and l, which
// attend_shared_join adds up with the other pieces and with what each sequence has
// behind the prefix.
//
// What bounds it.  One pass over K and V serves up to 256 rows (two tiles of 128), so
// up to about 250 rows a KV head it is HBM that does (4 bytes a token, dim and KV
// head in bf16 against 4 rows flops), and above that the tensor cores and the
// exponentials: a tile of 128 rows by 128 tokens of 128 dims is 1024 cycles of MMA
// and 1024 of ex2.
//
// Layout.  A block per SM, whose roles are warps:
//   0 - 3, 4 - 7  softmax of the first and the second tile of rows: a thread has a
//                 row, as tensor memory does
//   8             issues the MMAs
//   9 - 12        bring rows into shared memory: K and V tiles in a ring of slots,
//                 [64 dims][tokens][128 bytes] with the 128-byte swizzle, which is
//                 K-major for S and N-major for O, so V needs no transposing
// Tensor memory holds, for each tile of rows, S (one column a token; P takes the
// place of its first half as 16-bit pairs, the A operand of O's MMAs) and O.
// While one tile of rows is in its softmax the other's MMAs run.  Its pages are of
// any size, so rows come by 16-byte copies from wherever they lie.
//
// Rounding.  Operands are bf16 over bf16 caches under bf16 queries, else fp16:
//   a query of bf16 is brought to [2^14, 2^15) by a power of two a row, exact down to
//   2^-29 of its largest value;
//   Q8_0 and Q4_0 values are rounded to fp16 once, and F32 and BF16 ones too, each
//   group of tokens (a warp's 32 or 16) times a power of two that brings its largest
//   value below 2^15.  K's power multiplies the group's scores, V's is added to their
//   exponent, relative to the largest so far, and O carries that one;
//   probabilities are rounded to the operand type once, as the outputs are.  m may lag
//   behind the maximum by 2^8 before O is brought up to date, so fp16 probabilities
//   reach 2^15 and keep their bits down to 2^-21 of the largest.
// Sums are fp32.  An MMA truncates its sums, so O leaves tensor memory every
// kRunTokens tokens.
#pragma once

#include "attention_kernel.cuh"
#include "tc.cuh"

constexpr int kPrefixRows = 128;                  // of a tile
constexpr int kPrefixThreads = 13 * 32;
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
    float scale;                   // scores times log2 e
    unsigned long long page_mul;
    bool q_wide;                   // rows of q on 16 bytes
    float *part;                   // [slots][streams * 128][head_dim]
    float2 *part_ml;               // [slots][streams * 128]
    int *count;                    // of the call behind it, to be zeroed
    int counts;
    int *err;
    int device;
};

// Tokens of a tile: S and O of two tiles of rows fit tensor memory's 512 columns
// up to 192 dims.
constexpr int prefix_tile(int hd) { return hd <= 128 ? 128 : 64; }
constexpr int prefix_streams(int hd) { return hd <= 192 ? 2 : 1; }
constexpr int prefix_chunks(int hd) { return (hd + 63) / 64; }
constexpr int prefix_query_bytes(int hd) { return prefix_chunks(hd) * kPrefixRows * 128; }
constexpr int prefix_slot_bytes(int hd) { return prefix_chunks(hd) * prefix_tile(hd) * 128; }
constexpr int prefix_slots(int hd) {
    const int n = (222 * 1024 - prefix_streams(hd) * prefix_query_bytes(hd)) / prefix_slot_bytes(hd);
    return n < 8 ? n : 8;
}
// How the blocks share the units (a tile of tokens of one item), item by item.
struct PrefixRanges {
    int tiles;                     // of an item
    unsigned total, blocks, each, longer;
};
__host__ __device__ inline PrefixRanges prefix_ranges(int items, long long length, int tile, int blocks) {
    PrefixRanges r;
    r.tiles = (int)((length + tile - 1) / tile);
    r.total = (unsigned)items * (unsigned)r.tiles;
    r.blocks = r.total < (unsigned)blocks ? r.total : (unsigned)blocks;
    r.each = r.blocks ? r.total / r.blocks : 0;
    r.longer = r.total - r.each * r.blocks;
    return r;
}
__host__ __device__ inline unsigned prefix_block_of(const PrefixRanges &r, unsigned unit) {
    const unsigned split = r.longer * (r.each + 1);
    return unit < split ? unit / (r.each + 1) : r.longer + (unit - split) / r.each;
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

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }      // e in -126 .. 127

template <int kCache, int HD, bool kBf16>
__global__ void __launch_bounds__(kPrefixThreads, 1) prefix_kernel(const PrefixParams p) {
    constexpr int TN = prefix_tile(HD), GT = TN / 4, kChunks = prefix_chunks(HD), kSlots = prefix_slots(HD);
    constexpr int kQueryBytes = prefix_query_bytes(HD), kSlotBytes = prefix_slot_bytes(HD), kMaxStreams = prefix_streams(HD);
    constexpr int kRunTiles = kRunTokens / TN, kTileRing = 8;
    constexpr bool kRaw = (kCache == DTYPE_BF16 && kBf16) || kCache == DTYPE_F16;      // rows are copied as they are
    constexpr bool kQuant = kCache == DTYPE_Q8_0 || kCache == DTYPE_Q4_0;
    constexpr float kBias = kBf16 ? 0.0f : 7.0f, kLag = 8.0f;
    // fp32 += A B, both K-major for S; B's rows are the product's K for O
    constexpr uint32_t kFormat = (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(kPrefixRows >> 4) << 24);
    constexpr uint32_t kIdescS = kFormat | ((uint32_t)(TN >> 3) << 17), kIdescO = kFormat | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[kSlots], empty[kSlots], q_full, s_full[2], p_ready[2], o_full[2], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int s_abort;
    __shared__ float qmul[2][2][kPrefixRows];                     // [item's parity][tile of rows]
    __shared__ uint32_t counts[kTileRing][4];                     // tokens of a group that count
    __shared__ float k_up[kTileRing][4];                          // a group's keys are the operand's times this
    __shared__ int v_up[kTileRing][4];                            // and its values times 2 to this
    volatile int *const abort_flag = &s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();
    pdl_wait();
    const long long length = prefix_length(p, blockIdx.x == 0 && threadIdx.x == 0);
    for (int i = blockIdx.x * kPrefixThreads + threadIdx.x; i < p.counts; i += gridDim.x * kPrefixThreads) p.count[i] = 0;
    const PrefixRanges r = prefix_ranges(p.items, length, TN, p.blocks);
    if (blockIdx.x >= r.blocks) return;
    const unsigned lo = blockIdx.x * r.each + min(blockIdx.x, r.longer), hi = lo + r.each + (blockIdx.x < r.longer ? 1 : 0);
    const int item0 = (int)(lo / (unsigned)r.tiles), tile0 = (int)(lo - (unsigned)item0 * r.tiles), units = (int)(hi - lo);
    auto fail = [&]() {
        *abort_flag = 1;
        atomicOr(p.err, 2);
    };
    // Tiles of rows of an item.
    auto streams_of = [&](int item) { return min(p.streams, (p.rows - (item % p.row_sets) * p.streams * kPrefixRows + kPrefixRows - 1) / kPrefixRows); };
    // Whether a unit is the last of its item in this block, or the last of a run.
    auto last_of_item = [&](int n, int tile) { return n + 1 == units || tile + 1 == r.tiles; };

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(full + s, 4);
            mbar_init(empty + s, 1);
        }
        mbar_init(&q_full, 4);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_ready + i, 4);
            mbar_init(o_full + i, 1);
        }
        mbar_init(&done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t s_col[2] = {tmem, tmem + TN}, o_col[2] = {tmem + kMaxStreams * TN, tmem + kMaxStreams * TN + HD};
    uint8_t *const slots = smem + kMaxStreams * kQueryBytes;

    if (warp < 8) {
        // ------------------------------------------------------- softmax --
        const int i = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = s_col[i] + lanes, o_at = o_col[i] + lanes;
        float m = -INFINITY, l = 0.0f, qm = 0.0f;                 // of the run
        float m_item = -INFINITY, l_item = 0.0f;                  // of the item's runs before it
        int e_run = -1000, item = item0, tile = tile0, run = 0;
        uint32_t turn = 0, o_turn = 0;                            // tiles and runs of this tile of rows
        bool first_run = true;
        for (int n = 0; n < units; ++n) {
            const bool last = last_of_item(n, tile);
            if (i < streams_of(item)) {
                if (!wait_bounded(s_full + i, turn & 1, abort_flag)) {
                    if (lane == 0) fail();
                    break;
                }
                ++turn;
                tc_fence_after();
                const int ring = n % kTileRing;
                if (run == 0 && first_run) qm = qmul[(item - item0) & 1][i][row];
                uint32_t word[4];
                bool whole = true;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    word[g] = counts[ring][g];
                    whole = whole && word[g] == (GT == 32 ? 0xffffffffu : 0xffffu);
                }
                float qg[4];
                int eg[4], e_tile = -1000;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    qg[g] = kRaw ? qm : fmaxf(qm * k_up[ring][g], 1.2e-38f);
                    eg[g] = kRaw ? 0 : v_up[ring][g];
                    e_tile = max(e_tile, eg[g]);
                }
                // Scores of groups a and b, -inf where a token does not count.
                float s[2][GT];
                auto load = [&](int a) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) tmem_load<GT>(s_at + (a + k) * GT, reinterpret_cast<uint32_t *>(s[k]));
                    tmem_ld_wait();
                    if (!whole) {
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int j = 0; j < GT; ++j)
                                if (!((word[a + k] >> j) & 1)) s[k][j] = -INFINITY;
                    }
                };
                float top = -INFINITY;
                auto maximum = [&](int a) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float t0 = s[k][0], t1 = s[k][1];
#pragma unroll
                        for (int j = 2; j < GT; j += 2) {
                            t0 = fmaxf(t0, s[k][j]);
                            t1 = fmaxf(t1, s[k][j + 1]);
                        }
                        top = fmaxf(top, fmaxf(t0, t1) * qg[a + k]);
                    }
                };
                load(2);
                maximum(2);
                load(0);
                maximum(0);
                // ---- the reference, and O in its units ----
                const bool grew = top > m + kLag || (m == -INFINITY && top > m), up = !kRaw && e_tile > e_run;
                if (__any_sync(0xffffffffu, grew) || up) {
                    const float mn = fmaxf(m, top);
                    float f = mn == -INFINITY ? 1.0f : attn_exp2(m - mn);
                    l *= f;
                    m = mn;
                    if (up) {
                        if (run > 0) f *= pow2(max(e_run - e_tile, -126));
                        e_run = e_tile;
                    }
                    if (run > 0) {
                        // (S is behind the product of the tile before: O is at rest)
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            float o[32];
                            tmem_load<32>(o_at + c, reinterpret_cast<uint32_t *>(o));
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] *= f;
                            tmem_store<32>(o_at + c, reinterpret_cast<uint32_t *>(o));
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : kBias - m;
                auto probabilities = [&](int a) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int d = kRaw ? 0 : max(eg[a + k] - e_run, -100);
                        const float at = kRaw ? ref : ref + (float)d;
                        uint32_t w[GT / 2];
                        float sum[2] = {0.0f, 0.0f};
#pragma unroll
                        for (int j = 0; j < GT; j += 2) {
                            const float x = attn_exp2(fmaf(s[k][j], qg[a + k], at)), y = attn_exp2(fmaf(s[k][j + 1], qg[a + k], at));
                            sum[0] += x;
                            sum[1] += y;
                            w[j / 2] = pack16<kBf16>(x, y);
                        }
                        l += kRaw ? sum[0] + sum[1] : (sum[0] + sum[1]) * pow2(-d);
                        tmem_store<GT / 2>(s_at + (a + k) * (GT / 2), w);
                    }
                };
                probabilities(0);
                load(2);
                probabilities(2);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready + i);
                if (++run == kRunTiles || last) {
                    // ---- the run's O, added to the item's ----
                    if (!wait_bounded(o_full + i, o_turn & 1, abort_flag)) {
                        if (lane == 0) fail();
                        break;
                    }
                    ++o_turn;
                    tc_fence_after();
                    m -= kBias;
                    const size_t at = ((size_t)(blockIdx.x + item) * p.streams + i) * kPrefixRows + row;
                    float *to = p.part + at * HD;
                    const float top_ml = fmaxf(m, m_item), ref_ml = top_ml == -INFINITY ? 0.0f : top_ml;
                    const float w0 = first_run || l_item == 0.0f ? 0.0f : l_item * attn_exp2(m_item - ref_ml);
                    const float w1 = l == 0.0f ? 0.0f : l * attn_exp2(m - ref_ml), sum = w0 + w1;
                    const float f0 = sum == 0.0f ? 0.0f : w0 / sum;
                    const float f1 = l == 0.0f ? 0.0f : (w1 / sum) / l * (kRaw ? 1.0f : pow2(min(max(e_run, -126), 127)));
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
                        tmem_load<32>(o_at + c, reinterpret_cast<uint32_t *>(o));
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (l != 0.0f) y = make_float4(o[j] * f1, o[j + 1] * f1, o[j + 2] * f1, o[j + 3] * f1);
                            if (!first_run) {
                                const float4 x = *reinterpret_cast<const float4 *>(to + c + j);
                                y = make_float4(fmaf(x.x, f0, y.x), fmaf(x.y, f0, y.y), fmaf(x.z, f0, y.z), fmaf(x.w, f0, y.w));
                            }
                            *reinterpret_cast<float4 *>(to + c + j) = y;
                        }
                    }
                    tc_fence_before();
                    m_item = top_ml;
                    l_item = sum;
                    if (last) p.part_ml[at] = make_float2(m_item, l_item);
                    first_run = last;
                    m = -INFINITY;
                    l = 0.0f;
                    e_run = -1000;
                    run = 0;
                }
            }
            if (++tile == r.tiles) {
                tile = 0;
                ++item;
            }
        }
    } else if (warp == 8) {
        // ---------------------------------------------------------- MMAs --
        if (lane == 0) {
            uint32_t p_turn[2] = {0, 0};
            int item = item0, tile = tile0, run = 0;
            auto scores = [&](int i, int slot) {
                const uint32_t q = saddr(smem) + i * kQueryBytes, k = saddr(slots) + slot * kSlotBytes;
#pragma unroll
                for (int j = 0; j < HD / 16; ++j)
                    umma_bf16(s_col[i], sw128_desc(q + (j / 4) * (kPrefixRows * 128) + (j % 4) * 32),
                              sw128_desc(k + (j / 4) * (TN * 128) + (j % 4) * 32), kIdescS, j > 0);
                umma_commit(s_full + i);
            };
            auto wait_full = [&](int index) { return wait_bounded(full + index % kSlots, (index / kSlots) & 1, abort_flag); };
            bool ok = wait_bounded(&q_full, 0, abort_flag) && wait_full(0);
            if (ok) {
                tc_fence_after();
                for (int i = 0; i < streams_of(item); ++i) scores(i, 0);
                umma_commit(empty);
            }
            for (int n = 0; ok && n < units; ++n) {
                const bool last = last_of_item(n, tile), flush = run + 1 == kRunTiles || last;
                const int now = streams_of(item), next_item = tile + 1 == r.tiles ? item + 1 : item;
                const int next = n + 1 < units ? streams_of(next_item) : 0;
                const int vs = (2 * n + 1) % kSlots, ks = (2 * n + 2) % kSlots;
                bool ready = false;
                for (int i = 0; ok && i < max(now, next); ++i) {
                    if (i < now) {
                        ok = wait_bounded(p_ready + i, p_turn[i]++ & 1, abort_flag) && (i > 0 || wait_full(2 * n + 1));
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t v = saddr(slots) + vs * kSlotBytes;
#pragma unroll
                        for (int j = 0; j < TN / 16; ++j)
                            umma_ts(o_col[i], s_col[i] + 8 * j, sw128_desc_mn(v + j * 2048, TN * 128), kIdescO, run > 0 || j > 0);
                        if (flush) umma_commit(o_full + i);
                        if (i + 1 == now) umma_commit(empty + vs);
                    }
                    if (i < next) {
                        if (!ready) {
                            if (next_item != item) ok = wait_bounded(&q_full, (next_item - item0) & 1, abort_flag);
                            ok = ok && wait_full(2 * n + 2);
                            if (!ok) break;
                            tc_fence_after();
                            ready = true;
                        }
                        scores(i, ks);
                        if (i + 1 == next) umma_commit(empty + ks);
                    }
                }
                run = flush ? 0 : run + 1;
                if (++tile == r.tiles) {
                    tile = 0;
                    ++item;
                }
            }
            if (!ok) fail();
            umma_commit(&done);
            (void)wait_bounded(&done, 0, nullptr);
        }
        __syncwarp();
    } else {
        // ----------------------------------------------------- producers --
        const int w = warp - 9;                                   // its tokens: GT w .. of a tile, and rows 32 w .. of the query
        constexpr int kAhead = kRaw ? kSlots - 2 : 0;             // slots whose copies are on their way
        const int total = 2 * units;
        int signalled = 0;                                        // slots that this warp has filled
        bool ok = true;
        auto signal = [&](int index) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + index % kSlots);
        };
        auto drain = [&](int issued) {
            if constexpr (kRaw) copies_wait<0>();
            for (; signalled < issued; ++signalled) signal(signalled);
        };
        int item = item0, tile = tile0;
        unsigned row16 = 0, page16 = 0;                           // of token `lane` of the tile: its row, and its page
        int page_slot = 0;
        uint32_t valid = 0;
        int entry = -1, slot = 0;
        auto fetch = [&](int t) {                                 // looks the tokens of a tile up
            const long long tok = (long long)t * TN + w * GT + lane;
            entry = -1;
            if (lane < GT && tok < length) {
                int pg = (int)(((unsigned long long)(unsigned)tok * p.page_mul) >> 32);
                slot = (int)tok - pg * p.l.page_size;
                if (slot < 0) {
                    --pg;
                    slot += p.l.page_size;
                }
                entry = __ldg(p.table + pg);
            }
        };
        fetch(tile);
        for (int n = 0; ok && n < units; ++n) {
            const int kh = item / p.row_sets;
            if (n == 0 || tile == 0) {
                // ---- the item's queries ----
                if (n > 0) {
                    drain(2 * n);
                    const int index = 2 * n - 2;                  // the last scores of the item before
                    if (!wait_bounded(empty + index % kSlots, (index / kSlots) & 1, abort_flag)) {
                        if (lane == 0) fail();
                        break;
                    }
                }
                const int row = w * 32 + lane, swz = row & 7;
                for (int i = 0; i < streams_of(item); ++i) {
                    const int at = ((item % p.row_sets) * p.streams + i) * kPrefixRows + row;
                    const bool there = at < p.rows;
                    const int seq = there ? at / p.group : 0;
                    const long long from = seq * p.q_ss + (long long)(kh * p.group + (there ? at - seq * p.group : 0)) * p.q_hs;
                    uint8_t *to = smem + i * kQueryBytes + row * 128;
                    const bool convert = !kBf16 && p.io == DTYPE_BF16;
                    const uint16_t *src = static_cast<const uint16_t *>(p.q) + from;
                    auto piece = [&](int c, uint32_t (&x)[4]) {
                        uint4 u = make_uint4(0, 0, 0, 0);
                        if (there && p.q_wide) {
                            u = __ldg(reinterpret_cast<const uint4 *>(src) + c);
                        } else if (there) {
                            uint16_t h[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) h[j] = __ldg(src + 8 * c + j);
                            memcpy(&u, h, sizeof u);
                        }
                        const uint32_t sign = p.scale < 0.0f ? 0x80008000u : 0u;
                        x[0] = u.x ^ sign, x[1] = u.y ^ sign, x[2] = u.z ^ sign, x[3] = u.w ^ sign;
                    };
                    float up = 1.0f, mul = fmaxf(fabsf(p.scale), 1.2e-38f);
                    if (convert) {
                        uint32_t top = 0;                         // magnitudes are ordered like their bits
#pragma unroll 4
                        for (int c = 0; c < HD / 8; ++c) {
                            uint32_t x[4];
                            piece(c, x);
#pragma unroll
                            for (int j = 0; j < 4; ++j) top = max(top, max(x[j] & 0x7fffu, (x[j] >> 16) & 0x7fffu));
                        }
                        if (top > 0 && top < 0x7f80u) {
                            const int e = min(141 - (int)(top >> 7), 126);        // the largest goes to [2^14, 2^15)
                            up = pow2(e);
                            mul = fmaxf(mul * pow2(-e), 1.2e-38f);
                        }
                    }
#pragma unroll 4
                    for (int c = 0; c < HD / 8; ++c) {
                        uint32_t x[4];
                        piece(c, x);
                        if (convert) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                x[j] = half2_bits(__floats2half2_rn(__uint_as_float(x[j] << 16) * up, __uint_as_float(x[j] & 0xffff0000u) * up));
                        }
                        *reinterpret_cast<uint4 *>(to + (c / 8) * (kPrefixRows * 128) + (((c & 7) ^ swz) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                    qmul[(item - item0) & 1][i][row] = mul;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full);
            }
            // ---- where the tile's tokens are ----
            const bool found = (unsigned)entry < (unsigned)p.l.num_pages, wanted = lane < GT && (long long)tile * TN + w * GT + lane < length;
            page16 = (found ? (unsigned)entry : 0u) * (unsigned)(p.l.page_bytes >> 4);
            page_slot = slot;
            row16 = page16 + (unsigned)(slot * (p.l.row_bytes >> 4));
            valid = __ballot_sync(0xffffffffu, found && wanted);
            if (wanted && !found) atomicOr(p.err, kErrCache);
            if (n + 1 < units) fetch(tile + 1 == r.tiles ? 0 : tile + 1);
            const uint8_t *head = p.l.pages + (unsigned long long)kh * p.l.chunk_bytes;
            const int ring = n % kTileRing;

            // ---- K, then V ----
#pragma unroll 1
            for (int half = 0; ok && half < 2; ++half) {
                const int index = 2 * n + half;
                if (!wait_bounded(empty + index % kSlots, ((index / kSlots) & 1) ^ 1, abort_flag)) {
                    if (lane == 0) fail();
                    ok = false;
                    break;
                }
                uint8_t *const to = slots + (index % kSlots) * kSlotBytes;
                if constexpr (kRaw) {
                    constexpr int PR = HD / 8;                    // 16-byte pieces of a row
                    const uint8_t *from = head + (half ? p.l.v_off : 0);
                    const uint32_t dst = saddr(to);
#pragma unroll 8
                    for (int j = 0; j < GT * PR / 32; ++j) {
                        const int k = 32 * j + lane, t = k / PR, c = k - t * PR, row = w * GT + t;
                        const unsigned at = __shfl_sync(0xffffffffu, row16, t) + c;
                        copy_or_zero<16>(dst + (c >> 3) * (TN * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                                         from + ((unsigned long long)at << 4), (valid >> t) & 1);
                    }
                    if (half == 0 && lane == 0) counts[ring][w] = valid;
                    copies_commit();
                    if (signalled + kAhead <= index) {
                        copies_wait<kAhead>();
                        signal(signalled++);
                    }
                }
                (void)kQuant;
                (void)page_slot;
                (void)k_up;
                (void)v_up;
            }
            if (++tile == r.tiles) {
                tile = 0;
                ++item;
            }
        }
        if (ok) drain(total);
        else if constexpr (kRaw) copies_wait<0>();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int kCache, int HD, bool kBf16>
cudaError_t prefix_launch(const PrefixParams &p, cudaStream_t st) {
    constexpr size_t kBytes = 1024 + (size_t)prefix_streams(HD) * prefix_query_bytes(HD) + (size_t)prefix_slots(HD) * prefix_slot_bytes(HD);
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = attn_allow(prefix_kernel<kCache, HD, kBf16>, kBytes, p.device, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(prefix_kernel<kCache, HD, kBf16>, dim3(p.blocks), dim3(kPrefixThreads), kBytes, st, p);
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
cudaError_t prefix_run_bf16(const PrefixParams &p, cudaStream_t st);
cudaError_t prefix_run_f16(const PrefixParams &p, cudaStream_t st);
