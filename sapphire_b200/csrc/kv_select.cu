// kv_select.cu - pages chosen by a cheap score (include/sapphire_attention.h):
// bounds of every page's keys, kept beside the cache, and the selection of the
// pages that a new token attends to.
//
// Mathematics.  lo_d <= k_d <= hi_d for a page's keys gives q . k <= sum_d max(q_d
// hi_d, q_d lo_d), the most that one of its tokens could score.  Bounds and query
// are rounded to signed bytes (the bounds outwards), so the sum is a whole number
// below 2^23, the same in any order, and a selection does not depend on how a
// machine adds; what stays in fp32 is one product with each scale.
//
// As a product: a positive query value meets the upper bound and a negative one
// the lower, so a page's row [hi | lo] times the column [max(q, 0) | min(q, 0)] is
// the sum, an integer MMA of 16 pages by 8 query heads.
#include <algorithm>

#include "attention.cuh"

namespace {

constexpr float kMinNormal = 1.17549435e-38f;         // 2^-126

// max / 127 and its reciprocal, both 0 where the first is no normal number.
__device__ __forceinline__ float unit_of(float top, float &r) {
    const float s = __fdiv_rn(top, 127.0f);
    if (s < kMinNormal) {
        r = 0.0f;
        return 0.0f;
    }
    r = __frcp_rn(s);
    return s;
}

// ----------------------------------------------------------------- bounds --
// A block takes one KV head of one page.  A lane holds 8 dims of a row and walks
// down the page's rows, kRows loads in flight; the rows of a warp and the warps
// are joined at the end.  Every key of the page is read, so its bounds need no
// bounds before them: a page that a step adds one token to is read again, 16
// tokens of 256 bytes for one (8 KV heads of 32 sequences: 1 MB).
// A step is a chain of latencies (position, slot, rows, joining): 6 to 9 us for 0.4 to
// 1.2 MB.  A prompt of 20000 tokens of Q8_0 on 8 KV heads of 128 takes 18 us for 21 MB
// of keys (3 at HBM's rate), one warp to a page: unpacking and the chain of its loads.
// More rows in flight and several heads in a block gained nothing.
constexpr int kUnit = 8, kRows = 4, kMaxWarps = 8;

struct SummaryParams {
    KvLayout l;
    KvRows r;                     // (k and v unused)
    uint8_t *summary;
    unsigned long long summary_bytes;
    int *err;
};

template <int kCache>
struct KeyType {
    using type = float;
};
template <>
struct KeyType<DTYPE_BF16> {
    using type = __nv_bfloat16;
};
template <>
struct KeyType<DTYPE_F16> {
    using type = __half;
};

// Eight keys of a row as they lie in memory, and their value.
template <int kCache>
struct KeyUnit {
    static constexpr bool kQuant = kCache == DTYPE_Q8_0 || kCache == DTYPE_Q4_0;
    using T = typename KeyType<kCache>::type;
    Raw8<T> x;
    uint32_t w[2];
    float d;
    // u: the unit of the row; nb: blocks of a quantised row
    __device__ __forceinline__ void load(const uint8_t *row, const float *scales, int u, int nb) {
        if constexpr (kQuant) {
            const int word = 2 * (u & 3) * nb + (u >> 2);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                w[j] = kCache == DTYPE_Q8_0 ? reinterpret_cast<const uint32_t *>(row)[word + j * nb] : reinterpret_cast<const uint16_t *>(row)[word + j * nb];
            d = scales[u >> 2];
        } else {
            x.load(reinterpret_cast<const T *>(row) + u * kUnit, true);
        }
    }
    __device__ __forceinline__ void get(float (&v)[kUnit]) const {
        if constexpr (kQuant) {
#pragma unroll
            for (int j = 0; j < kUnit; ++j) {
                const uint32_t q = kCache == DTYPE_Q8_0 ? __byte_perm(w[j / 4], 0x4b000000u, 0x7440 + (j & 3))
                                                        : ((w[j / 4] >> (4 * (j & 3))) & 15u) | 0x4b000000u;
                v[j] = __fmul_rn(__fadd_rn(__uint_as_float(q), kCache == DTYPE_Q8_0 ? -8388736.0f : -8388616.0f), d);
            }
        } else {
            x.get(v);
        }
    }
};

template <int kCache>
__global__ void __launch_bounds__(kMaxWarps * 32) kv_summary_kernel(const SummaryParams p) {
    extern __shared__ float part[];                               // [warp][hi, lo][dim], of several warps
    pdl_trigger();
    pdl_wait();
    const int h = blockIdx.y, page_size = p.l.page_size;
    // ---- which page: candidates are numbered so that sequence s has at least as
    //      many as its new tokens touch pages: floor(cu[s] / page_size) + 2 s on ----
    int s = blockIdx.x, j = 0, n = 1;
    if (p.r.cu_tokens) {
        // (Lanes look at 32 places between at a time: a load for each factor of 33.)
        int lo = 0, hi = p.r.sequences;                           // the sequence is in [lo, hi)
        while (hi - lo > 1) {
            const int gap = (hi - lo + 32) / 33, at = lo + ((int)threadIdx.x % 32 + 1) * gap;
            const bool before = at < hi && (long long)(__ldg(p.r.cu_tokens + at) / page_size) + 2ll * at <= (long long)blockIdx.x;
            const int steps = __popc(__ballot_sync(0xffffffffu, before));
            hi = min(hi, lo + (steps + 1) * gap);
            lo += steps * gap;
        }
        s = lo;
        const int cu = __ldg(p.r.cu_tokens + s);
        n = __ldg(p.r.cu_tokens + s + 1) - cu;
        const long long at = (long long)blockIdx.x - cu / page_size - 2ll * s;
        if (at < 0 || at > n) return;
        j = (int)at;
    }
    const long long begin = p.r.start ? __ldg(p.r.start + s) : 0, end = begin + n;
    const long long page = (begin >= 0 ? begin / page_size : 0) + j;
    if (n <= 0 || page * page_size >= end) return;
    if (begin < 0 || page >= p.r.table_stride) {
        if (threadIdx.x == 0) atomicOr(p.err, kErrCache);
        return;
    }
    const int id = __ldg(p.r.page_table + (long long)s * p.r.table_stride + page);
    if (id < 0 || id >= p.l.num_pages) {
        if (threadIdx.x == 0) atomicOr(p.err, kErrCache);
        return;
    }
    const int rows = (int)min((long long)page_size, end - page * page_size);

    // ---- this lane's rows ----
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int units = p.l.head_dim / kUnit, group = 32 / units, nb = p.l.head_dim / 32;
    const int row0 = lane / units, u = lane - row0 * units;
    const uint8_t *chunk = p.l.pages + (unsigned long long)id * p.l.page_bytes + (unsigned long long)h * p.l.chunk_bytes;
    const float *scales = reinterpret_cast<const float *>(chunk + p.l.ks_off);
    float hi[kUnit], lo[kUnit];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
        hi[i] = -INFINITY;
        lo[i] = INFINITY;
    }
    const int step = group * warps;
    if (row0 < group) {
        for (int r = warp * group + row0; r < rows; r += kRows * step) {
            KeyUnit<kCache> x[kRows];
#pragma unroll
            for (int k = 0; k < kRows; ++k)
                if (r + k * step < rows) x[k].load(chunk + (long long)(r + k * step) * p.l.row_bytes, scales + (r + k * step) * p.l.scale_stride, u, nb);
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                if (r + k * step >= rows) continue;
                float v[kUnit];
                x[k].get(v);
#pragma unroll
                for (int i = 0; i < kUnit; ++i) {
                    hi[i] = fmaxf(hi[i], v[i]);
                    lo[i] = fminf(lo[i], v[i]);
                    bad = bad || !(fabsf(v[i]) < INFINITY);
                }
            }
        }
    }
    // ---- the rows of the warp, and the warps ----
    for (int k = 1; k < group; ++k) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            const float a = __shfl_sync(0xffffffffu, hi[i], (u + k * units) & 31), b = __shfl_sync(0xffffffffu, lo[i], (u + k * units) & 31);
            if (row0 == 0) {
                hi[i] = fmaxf(hi[i], a);
                lo[i] = fminf(lo[i], b);
            }
        }
    }
    if (warps > 1) {
        if (row0 == 0) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) {
                part[(2 * warp) * p.l.head_dim + u * kUnit + i] = hi[i];
                part[(2 * warp + 1) * p.l.head_dim + u * kUnit + i] = lo[i];
            }
        }
        bad = __syncthreads_or(bad);
        if (warp > 0) return;
        if (row0 == 0) {
            for (int w = 1; w < warps; ++w)
#pragma unroll
                for (int i = 0; i < kUnit; ++i) {
                    hi[i] = fmaxf(hi[i], part[(2 * w) * p.l.head_dim + u * kUnit + i]);
                    lo[i] = fminf(lo[i], part[(2 * w + 1) * p.l.head_dim + u * kUnit + i]);
                }
        }
    } else {
        bad = __any_sync(0xffffffffu, bad);
    }
    float top = 0.0f;
    if (row0 == 0) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) top = fmaxf(top, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float r, unit = unit_of(top, r);
    uint32_t code[2][2] = {};
    if (bad) {
        unit = INFINITY;
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            const int a = max(-127, min(127, __float2int_ru(__fmul_rn(hi[i], r)))), b = max(-127, min(127, __float2int_rd(__fmul_rn(lo[i], r))));
            code[0][i / 4] |= (uint32_t)(a & 255) << (8 * (i & 3));
            code[1][i / 4] |= (uint32_t)(b & 255) << (8 * (i & 3));
        }
    }
    uint8_t *to = p.summary + (unsigned long long)id * p.summary_bytes;
    if (row0 == 0) {
        uint8_t *codes = to + (unsigned long long)h * 2 * p.l.head_dim + u * kUnit;
        *reinterpret_cast<uint2 *>(codes) = make_uint2(code[0][0], code[0][1]);
        *reinterpret_cast<uint2 *>(codes + p.l.head_dim) = make_uint2(code[1][0], code[1][1]);
    }
    if (lane == 0) reinterpret_cast<float *>(to + (unsigned long long)p.l.kv_heads * 2 * p.l.head_dim)[h] = unit;
}

// -------------------------------------------------------------- selection --
// A cluster of 1 to 8 blocks takes one KV head of one sequence: each block scores
// a range of the pages, 16 a warp at a time, and keeps their keys (the scores'
// bits, ordered as whole numbers) in shared memory.  The smallest key that is in is
// found by digits of 8 bits below the keys' highest differing one, the counts
// of the cluster's blocks added through distributed shared memory; a round whose
// digit takes all its keys is the last.  Then each thread counts what it has in a
// range of neighbouring pages, and a sum over the threads before it gives the place
// of each, so the pages come out in order.
// What bounds it: 64 sequences of up to 512 pages, 8 KV heads of 128, take 27 us
// for 51 MB (8 at HBM's rate; DRAM 23 %, issue 35 %): the scores near HBM's rate while
// they last, before them the query's codes, after them three rounds of digits, each a
// barrier of the cluster, and the places.  One sequence of 128 pages takes 8 us, which
// are that chain.  So the first pages' bounds are on their way before the query is read,
// and page numbers a turn ahead of their use (28.5 -> 27 us).
constexpr int kSelThreads = 256, kSelWarps = kSelThreads / 32;
constexpr int kMaxCluster = 8, kMaxKeys = 32768;      // keys of a block: 128 KB
constexpr int kMaxGroup = 128;

struct SelectParams {
    const void *q;
    long long q_ss, q_hs;
    const uint8_t *summary;
    unsigned long long summary_bytes;
    const int *page_table, *lengths;
    int *selected, *selected_lengths;
    int io, num_pages, kv_heads, head_dim, group, page_size, table_stride, length_offset;
    int budget, first, last;
    int block_keys;                                   // room for keys of a block
    int *err;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The 32-bit word of block `rank` that lies where p lies in this one.
__device__ __forceinline__ uint32_t cluster_read(const void *p, uint32_t rank) {
    uint32_t at = (uint32_t)__cvta_generic_to_shared(p), v;
    asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float load_io(const void *q, int io, long long at) {
    return io == DTYPE_F32  ? __ldg(static_cast<const float *>(q) + at)
           : io == DTYPE_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(q)[at])
                              : __half2float(static_cast<const __half *>(q)[at]);
}

// Chunks of 64 bytes of a page's row [hi | lo].
template <int kChunks>
__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const SelectParams p) {
    constexpr int HD = 32 * kChunks, kStride = 2 * HD + 64;   // (rows of neighbouring columns on the other half of the banks)
    extern __shared__ __align__(16) uint8_t shared[];
    uint32_t *const keys = reinterpret_cast<uint32_t *>(shared);
    uint8_t *const qc = shared + (size_t)p.block_keys * 4;        // [columns][kStride]
    __shared__ float qt[kMaxGroup];
    __shared__ unsigned hist[2][256];
    __shared__ uint32_t range[2];                                 // least and largest key
    __shared__ uint32_t totals[2];                                // keys above the threshold, and at it
    __shared__ uint32_t found[4];                                 // the digit, what is still wanted, its count
    __shared__ unsigned long long warp_sum[kSelWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y, s = blockIdx.z;
    const uint32_t rank = cluster_rank(), blocks = cluster_size();
    pdl_trigger();
    pdl_wait();
    long long n = (long long)__ldg(p.lengths + s) + p.length_offset;
    const long long room = (long long)p.table_stride * p.page_size;
    if (n < 0 || n > room) {
        if (tid == 0 && rank == 0 && h == 0) atomicOr(p.err, kErrCache);
        n = n < 0 ? 0 : room;
    }
    const int pages = (int)((n + p.page_size - 1) / p.page_size);
    const int *table = p.page_table + (long long)s * p.table_stride;
    int *const out = p.selected + ((long long)s * p.kv_heads + h) * p.budget;
    if (tid == 0 && rank == 0 && h == 0) p.selected_lengths[s] = (int)(n - (long long)max(0, pages - p.budget) * p.page_size);
    if (pages <= p.budget) {                                      // (of the whole cluster)
        for (int i = rank * kSelThreads + tid; i < p.budget; i += blocks * kSelThreads) out[i] = i < pages ? __ldg(table + i) : -1;
        return;
    }
    for (int i = rank * kSelThreads + tid; i < p.first + p.last; i += blocks * kSelThreads)
        out[i < p.first ? i : p.budget - p.last + (i - p.first)] = __ldg(table + (i < p.first ? i : pages - p.last + (i - p.first)));
    const int wanted = p.budget - p.first - p.last, middle = pages - p.first - p.last;      // of these pages
    if (wanted == 0) return;

    // ---- this block's pages [begin, begin + mine) of the middle: page numbers are looked up
    //      a turn ahead, and the first turn's rows are on their way while the query is
    //      made codes ----
    const int per = (middle + (int)blocks - 1) / (int)blocks, begin = min((int)rank * per, middle), mine = min(per, middle - begin);
    const uint8_t *const codes = p.summary + (unsigned long long)h * 2 * HD;
    const unsigned long long scale_at = (unsigned long long)p.kv_heads * 2 * HD + 4ull * h;
    int ids[2];
    auto look = [&](int i0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) ids[k] = i0 + 8 * k + g < mine ? __ldg(table + p.first + begin + i0 + 8 * k + g) : -1;
    };
    // Lane (g, t) reads 16 bytes of each 64 of rows g and g + 8: as the order of dims is
    // the query's too, they are the MMA's fragments.
    uint4 a[2][kChunks];
    float d[2];
    bool ok[2];
    auto rows = [&](int i0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            ok[k] = (unsigned)ids[k] < (unsigned)p.num_pages;
            if (i0 + 8 * k + g < mine && !ok[k]) atomicOr(p.err, kErrCache);
            const uint8_t *row = codes + (unsigned long long)(ok[k] ? ids[k] : 0) * p.summary_bytes;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) a[k][c] = __ldg(reinterpret_cast<const uint4 *>(row + 64 * c) + t);
            d[k] = __ldg(reinterpret_cast<const float *>(p.summary + (unsigned long long)(ok[k] ? ids[k] : 0) * p.summary_bytes + scale_at));
        }
    };
    look(warp * 16);
    rows(warp * 16);
    // ---- the query's codes: columns of [max(c, 0) | min(c, 0)] ----
    const int columns = (p.group + 7) & ~7;
    for (int j = warp; j < columns; j += kSelWarps) {
        float x[kChunks], top = 0.0f;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            x[i] = j < p.group ? load_io(p.q, p.io, s * p.q_ss + (long long)(h * p.group + j) * p.q_hs + 32 * i + lane) : 0.0f;
            top = fabsf(x[i]) < INFINITY ? fmaxf(top, fabsf(x[i])) : INFINITY;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float r = 0.0f, unit = 0.0f;
        if (top < INFINITY) unit = unit_of(top, r);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = top < INFINITY ? (int)roundf(__fmul_rn(x[i], r)) : 0;
            qc[j * kStride + 32 * i + lane] = (uint8_t)max(c, 0);
            qc[j * kStride + HD + 32 * i + lane] = (uint8_t)min(c, 0);
        }
        if (lane == 0) qt[j] = unit;
    }
    hist[0][tid] = hist[1][tid] = 0;
    if (tid == 0) {
        range[0] = 0xffffffffu;
        range[1] = 0;
    }
    __syncthreads();

    // ---- scores of this block's pages [begin, begin + mine) of the middle ----
    uint32_t least = 0xffffffffu, most = 0;
    for (int i0 = warp * 16; i0 < mine; i0 += kSelWarps * 16) {
        if (i0 >= kSelWarps * 16) rows(i0);
        look(i0 + kSelWarps * 16);
        float best[2] = {-INFINITY, -INFINITY};
        for (int j0 = 0; j0 < p.group; j0 += 8) {
            int c[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < kChunks; ++k) {
                const uint4 b = *reinterpret_cast<const uint4 *>(qc + (j0 + g) * kStride + 64 * k + 16 * t);
                mma_s8(c, a[0][k].x, a[1][k].x, a[0][k].y, a[1][k].y, b.x, b.y);
                mma_s8(c, a[0][k].z, a[1][k].z, a[0][k].w, a[1][k].w, b.z, b.w);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (j0 + 2 * t + e >= p.group) continue;
                const float unit = qt[j0 + 2 * t + e];
                best[0] = fmaxf(best[0], __fmul_rn((float)c[e], unit));
                best[1] = fmaxf(best[1], __fmul_rn((float)c[2 + e], unit));
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            best[k] = fmaxf(best[k], __shfl_xor_sync(0xffffffffu, best[k], 1));
            best[k] = fmaxf(best[k], __shfl_xor_sync(0xffffffffu, best[k], 2));
            float score = d[k] == 0.0f ? 0.0f : d[k] < INFINITY ? __fmul_rn(best[k], d[k]) : INFINITY;
            if (!ok[k]) score = -INFINITY;                        // nothing there
            const uint32_t bits = __float_as_uint(__fadd_rn(score, 0.0f));       // one zero
            const uint32_t key = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
            if (t == 0 && i0 + 8 * k + g < mine) {
                keys[i0 + 8 * k + g] = key;
                least = min(least, key);
                most = max(most, key);
            }
        }
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
        atomicMin(range, least);
        atomicMax(range + 1, most);
    }
    if (blocks > 1) {
        cluster_barrier();
        for (uint32_t b = 0; b < blocks; ++b) {
            least = min(least, cluster_read(range, b));
            most = max(most, cluster_read(range + 1, b));
        }
    } else {
        __syncthreads();
        least = range[0];
        most = range[1];
    }

    // ---- the threshold: `low` is the smallest key that is in, of whose kind
    //      `ties` are (the first ones) ----
    const uint32_t span = most - least;
    int shift = max(0, 24 - __clz(span | 1));                     // the digit's lowest bit
    uint32_t low = 0, ties = wanted, same = 0;                    // above `least`; keys of the digits so far
    uint32_t prefix_shift = 32;
    for (int round = 0;; ++round) {
        unsigned *const my = hist[round & 1];
        for (int i = tid; i < mine; i += kSelThreads) {
            const uint32_t y = keys[i] - least;
            if (prefix_shift == 32 || (y >> prefix_shift) == (low >> prefix_shift)) atomicAdd(my + ((y >> shift) & 255), 1u);
        }
        unsigned count;
        if (blocks > 1) {
            cluster_barrier();
            count = 0;
            for (uint32_t b = 0; b < blocks; ++b) count += cluster_read(my + tid, b);
        } else {
            __syncthreads();
            count = my[tid];
        }
        hist[(round + 1) & 1][tid] = 0;               // (its readers are behind this round's barrier)
        // Keys of higher digits: a sum over the bins from the top.
        unsigned above = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_down_sync(0xffffffffu, above, o);
            if (lane + o < 32) above += v;
        }
        if (lane == 0) warp_sum[warp] = above;
        __syncthreads();
        for (int w = warp + 1; w < kSelWarps; ++w) above += (unsigned)warp_sum[w];
        if (above >= ties && above - count < ties) {              // of one thread
            found[0] = tid;
            found[1] = ties - (above - count);
            found[2] = count;
        }
        __syncthreads();
        low |= found[0] << shift;
        ties = found[1];
        same = found[2];
        if (same == ties || shift == 0) break;
        prefix_shift = shift;
        shift = max(0, shift - 8);
    }
    // Keys whose digits above `shift` are above low's are in; those that share
    // them are in where all are (same == ties), else the first `ties` of them.
    // ---- places ----
    const int each = (mine + kSelThreads - 1) / kSelThreads, i0 = min(tid * each, mine), i1 = min(i0 + each, mine);
    uint32_t over = 0, at = 0;
    for (int i = i0; i < i1; ++i) {
        const uint32_t y = (keys[i] - least) >> shift;
        over += y > low >> shift;
        at += y == low >> shift;
    }
    unsigned long long sum = (unsigned long long)over << 32 | at, before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = before;
    __syncthreads();
    unsigned long long all = 0;
    before -= sum;
    for (int w = 0; w < kSelWarps; ++w) {
        if (w < warp) before += warp_sum[w];
        all += warp_sum[w];
    }
    if (blocks > 1) {
        if (tid == 0) {
            totals[0] = (uint32_t)(all >> 32);
            totals[1] = (uint32_t)all;
        }
        cluster_barrier();
        for (uint32_t b = 0; b < rank; ++b) before += (unsigned long long)cluster_read(totals, b) << 32 | cluster_read(totals + 1, b);
    }
    uint32_t place_over = (uint32_t)(before >> 32), place_at = (uint32_t)before;
    for (int i = i0; i < i1; ++i) {
        const uint32_t y = (keys[i] - least) >> shift;
        const bool is_over = y > low >> shift, is_at = y == low >> shift;
        if (is_over || (is_at && place_at < ties)) out[p.first + place_over + min(place_at, ties)] = __ldg(table + p.first + begin + i);
        place_over += is_over;
        place_at += is_at;
    }
    if (blocks > 1) cluster_barrier();                // a block's shared memory lives until all have read it
}

size_t summary_bytes(const sapphire_kv_cache_t *c) {
    return (size_t)c->kv_heads * 2 * c->head_dim + (((size_t)c->kv_heads * 4 + 15) & ~(size_t)15);
}

template <int kChunks>
cudaError_t launch_select(const SelectParams &p, int sequences, int cluster, int device, cudaStream_t st) {
    const size_t bytes = (size_t)p.block_keys * 4 + (size_t)((p.group + 7) & ~7) * (64 * kChunks + 64);
    static std::atomic<unsigned long long> done{0};
    const unsigned long long bit = 1ull << (device & 63);
    if (!(done.load(std::memory_order_acquire) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kv_select_kernel<kChunks>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   kMaxKeys * 4 + kMaxGroup * (64 * kChunks + 64));
        if (e != cudaSuccess) return e;
        done.fetch_or(bit, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster, p.kv_heads, sequences);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kv_select_kernel<kChunks>, p);
}

}  // namespace

extern "C" SAPPHIRE_API size_t sapphire_kv_summary_bytes(const sapphire_kv_cache_t *cache) {
    return cache && sapphire_kv_page_bytes(cache) ? summary_bytes(cache) : 0;
}

extern "C" SAPPHIRE_API int sapphire_kv_summarise_device(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                                         void *summary, const sapphire_kv_args_t *a) {
    const char *who = "sapphire_kv_summarise_device";
    if (!ctx || !cache || !a) {
        LOG_ERROR("%s: NULL argument", who);
        return -1;
    }
    std::lock_guard<std::recursive_mutex> lk(ctx->exec_mutex);
    if (!ctx->initialized) {
        ctx_fail(ctx, who, "context not initialized");
        return -1;
    }
    SummaryParams p{};
    if (!kv_layout(ctx, who, cache, &p.l)) return -1;
    if (a->tokens < 0 || a->sequences < 0 || (!a->cu_tokens && a->tokens != a->sequences)) {
        ctx_fail(ctx, who, "%d tokens of %d sequences (without cu_tokens each has one)", a->tokens, a->sequences);
        return -1;
    }
    if (a->tokens == 0 || a->sequences == 0) return 0;
    if (a->table_stride <= 0) {
        ctx_fail(ctx, who, "table_stride must be positive");
        return -1;
    }
    if (!on_device(ctx, who, "pages", cache->pages) || !on_device(ctx, who, "summary", summary) ||
        !on_device(ctx, who, "page_table", a->page_table) ||
        (a->cu_tokens && !on_device(ctx, who, "cu_tokens", a->cu_tokens)) ||
        (a->start && !on_device(ctx, who, "start", a->start)))
        return -1;
    if ((uintptr_t)summary & 15) {
        ctx_fail(ctx, who, "the summary must be 16-byte aligned");
        return -1;
    }
    const long long candidates = a->cu_tokens ? a->tokens / cache->page_size + 2ll * a->sequences : a->sequences;
    if (candidates > INT32_MAX) {
        ctx_fail(ctx, who, "%d tokens of %d sequences are more than 2^31 pages", a->tokens, a->sequences);
        return -1;
    }
    p.r.cu_tokens = a->cu_tokens;
    p.r.start = a->start;
    p.r.page_table = a->page_table;
    p.r.tokens = a->tokens;
    p.r.sequences = a->sequences;
    p.r.table_stride = a->table_stride;
    p.summary = static_cast<uint8_t *>(summary);
    p.summary_bytes = summary_bytes(cache);
    p.err = ctx->d_err;
    AttnDevice g(ctx->device);
    // A warp for each 16 rows (its loads in flight), up to 8.
    int warps = 1;
    while (warps < kMaxWarps && warps * 16 < cache->page_size) warps *= 2;
    const dim3 grid((unsigned)candidates, cache->kv_heads), block(32 * warps);
    const size_t bytes = warps > 1 ? (size_t)warps * 2 * cache->head_dim * sizeof(float) : 0;
    cudaError_t e;
    switch (cache->dtype) {
        case DTYPE_F32: e = launch_pdl(kv_summary_kernel<DTYPE_F32>, grid, block, bytes, ctx->stream, p); break;
        case DTYPE_BF16: e = launch_pdl(kv_summary_kernel<DTYPE_BF16>, grid, block, bytes, ctx->stream, p); break;
        case DTYPE_F16: e = launch_pdl(kv_summary_kernel<DTYPE_F16>, grid, block, bytes, ctx->stream, p); break;
        case DTYPE_Q8_0: e = launch_pdl(kv_summary_kernel<DTYPE_Q8_0>, grid, block, bytes, ctx->stream, p); break;
        default: e = launch_pdl(kv_summary_kernel<DTYPE_Q4_0>, grid, block, bytes, ctx->stream, p); break;
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        ctx_fail(ctx, who, "launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}

extern "C" SAPPHIRE_API int sapphire_kv_select_device(kernel_context_t *ctx, const sapphire_kv_cache_t *cache,
                                                      const sapphire_kv_select_args_t *a) {
    const char *who = "sapphire_kv_select_device";
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
    if (!io_size(a->dtype)) {
        ctx_fail(ctx, who, "q must be F32, BF16 or F16");
        return -1;
    }
    if (a->heads <= 0 || a->heads % cache->kv_heads || a->heads / cache->kv_heads > kMaxGroup) {
        ctx_fail(ctx, who, "%d query heads over %d KV heads (at most %d to one)", a->heads, cache->kv_heads, kMaxGroup);
        return -1;
    }
    if (a->sequences < 0 || a->sequences > 65535) {
        ctx_fail(ctx, who, "sequences must be 0 to 65535");
        return -1;
    }
    if (a->sequences == 0) return 0;
    if (a->table_stride <= 0 || a->table_stride > kMaxCluster * kMaxKeys) {
        ctx_fail(ctx, who, "table_stride must be 1 to %d", kMaxCluster * kMaxKeys);
        return -1;
    }
    if (a->first < 0 || a->last < 1 || a->budget < 1 || (long long)a->first + a->last > a->budget) {
        ctx_fail(ctx, who, "a budget of %d pages with the first %d and the last %d (1 or more) always in it", a->budget, a->first, a->last);
        return -1;
    }
    if (!on_device(ctx, who, "summary", a->summary) || !on_device(ctx, who, "q", a->q) ||
        !on_device(ctx, who, "page_table", a->page_table) || !on_device(ctx, who, "lengths", a->lengths) ||
        !on_device(ctx, who, "selected", a->selected) || !on_device(ctx, who, "selected_lengths", a->selected_lengths))
        return -1;
    if ((uintptr_t)a->summary & 15) {
        ctx_fail(ctx, who, "the summary must be 16-byte aligned");
        return -1;
    }
    SelectParams p{};
    p.q = a->q;
    p.q_ss = a->q_seq_stride ? a->q_seq_stride : (long long)a->heads * cache->head_dim;
    p.q_hs = a->q_head_stride ? a->q_head_stride : cache->head_dim;
    p.summary = static_cast<const uint8_t *>(a->summary);
    p.summary_bytes = summary_bytes(cache);
    p.page_table = a->page_table;
    p.lengths = a->lengths;
    p.selected = a->selected;
    p.selected_lengths = a->selected_lengths;
    p.io = a->dtype;
    p.num_pages = cache->num_pages;
    p.kv_heads = cache->kv_heads;
    p.head_dim = cache->head_dim;
    p.group = a->heads / cache->kv_heads;
    p.page_size = cache->page_size;
    p.table_stride = a->table_stride;
    p.length_offset = a->length_offset;
    p.budget = a->budget;
    p.first = a->first;
    p.last = a->last;
    p.err = ctx->d_err;
    AttnDevice g(ctx->device);
    // Blocks of a cluster: as many as the GPU holds two on an SM of, where each
    // still has a turn of its warps (128 pages); more where the keys need the room.
    const long long items = (long long)a->sequences * cache->kv_heads;
    int cluster = 1;
    while (cluster < kMaxCluster && items * cluster * 2 <= 2 * sm_count(ctx->device) && a->table_stride > 128 * cluster) cluster *= 2;
    while (a->table_stride > (long long)cluster * kMaxKeys) cluster *= 2;
    p.block_keys = (((a->table_stride + cluster - 1) / cluster) + 3) & ~3;
    cudaError_t e;
    switch (cache->head_dim) {
        case 64: e = launch_select<2>(p, a->sequences, cluster, ctx->device, ctx->stream); break;
        case 96: e = launch_select<3>(p, a->sequences, cluster, ctx->device, ctx->stream); break;
        case 128: e = launch_select<4>(p, a->sequences, cluster, ctx->device, ctx->stream); break;
        case 192: e = launch_select<6>(p, a->sequences, cluster, ctx->device, ctx->stream); break;
        default: e = launch_select<8>(p, a->sequences, cluster, ctx->device, ctx->stream); break;
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        ctx_fail(ctx, who, "launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    return 0;
}
