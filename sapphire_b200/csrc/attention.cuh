// attention.cuh - what the rotary, paged-cache and attention sources share
// (include/sapphire_attention.h): element types, the cache's byte layout and
// the checks of arguments.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.cuh"
#include "../../include/sapphire_attention.h"

// Error-word bit of a page number, position or length outside the cache.
constexpr int kErrCache = 32;

// The bytes of a page (include/sapphire_attention.h): for each KV head a chunk
// [K rows | V rows | K scales | V scales].
struct KvLayout {
    uint8_t *pages;
    unsigned long long page_bytes;
    int num_pages, page_size, kv_heads, head_dim;
    int row_bytes;       // one row of codes or values
    int scale_stride;    // padded scales of a row (0: dense)
    int chunk_bytes;     // one KV head of a page
    int v_off;           // V rows inside a chunk
    int ks_off, vs_off;  // K and V scales inside a chunk
};

// Ragged rows (sapphire_kv_args_t).
struct KvRows {
    const int *cu_tokens, *start, *page_table;
    int tokens, sequences, table_stride;
    void *k, *v;
    long long k_ts, k_hs, v_ts, v_hs;
};

// Whether every row starts on `bytes` bytes.
inline bool rows_aligned(const void *p, long long ts, long long hs, size_t elem, int bytes = 16) {
    return (uintptr_t)p % bytes == 0 && (ts * (long long)elem) % bytes == 0 && (hs * (long long)elem) % bytes == 0;
}

// Fills `l` from the caller's cache; false (with the context's error set when
// ctx is given) if the shape is not supported.
bool kv_layout(kernel_context_t *ctx, const char *who, const sapphire_kv_cache_t *c, KvLayout *l);
// Whether p is device memory of the context's GPU (recorded as an error if not).
bool on_device(kernel_context_t *ctx, const char *who, const char *what, const void *p);

inline size_t io_size(tensor_dtype_t dt) { return dt == DTYPE_F32 ? 4 : (dt == DTYPE_BF16 || dt == DTYPE_F16) ? 2 : 0; }

// Restores the caller's device on scope exit.
struct AttnDevice {
    int prev = -1, dev;
    explicit AttnDevice(int d) : dev(d) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) cudaSetDevice(dev);
    }
    ~AttnDevice() {
        if (prev >= 0 && prev != dev) cudaSetDevice(prev);
    }
};

#ifdef __CUDACC__
template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) {
    return __bfloat162float(x);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) {
    return __half2float(x);
}
// One rounding, to nearest even.
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
    return __float2half_rn(x);
}

// kCount (8 or 4) consecutive values as they lie in memory, so that loads in
// flight hold no more registers than their bytes.
template <int kBytes>
struct RawWord {
    using type = uint4;
};
template <>
struct RawWord<8> {
    using type = uint2;
};
template <typename T, int kCount>
struct Raw {
    using Word = typename RawWord<kCount * sizeof(T)>::type;
    static constexpr int N = kCount * sizeof(T) / sizeof(Word);
    Word v[N];
    // wide: p is on 16 bytes (8 where that is all)
    __device__ __forceinline__ void load(const T *p, bool wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = reinterpret_cast<const Word *>(p)[i];
        } else {
            T t[kCount];
#pragma unroll
            for (int j = 0; j < kCount; ++j) t[j] = p[j];
            memcpy(v, t, sizeof v);
        }
    }
    __device__ __forceinline__ void store(T *p, bool wide) const {
        if (wide) {
#pragma unroll
            for (int i = 0; i < N; ++i) reinterpret_cast<Word *>(p)[i] = v[i];
        } else {
            T t[kCount];
            memcpy(t, v, sizeof v);
#pragma unroll
            for (int j = 0; j < kCount; ++j) p[j] = t[j];
        }
    }
    __device__ __forceinline__ void get(float (&x)[kCount]) const {
        T t[kCount];
        memcpy(t, v, sizeof v);
#pragma unroll
        for (int j = 0; j < kCount; ++j) x[j] = to_f32(t[j]);
    }
    __device__ __forceinline__ void set(const float (&x)[kCount]) {
        T t[kCount];
#pragma unroll
        for (int j = 0; j < kCount; ++j) t[j] = from_f32<T>(x[j]);
        memcpy(v, t, sizeof v);
    }
};
template <typename T>
using Raw8 = Raw<T, 8>;
#endif
