// prefix_bf16.cu - a shared prefix over BF16 pages (prefix_kernel.cuh).
#include "prefix_kernel.cuh"

cudaError_t prefix_run_bf16(const PrefixParams &p, cudaStream_t st) { return prefix_launch<DTYPE_BF16, true>(p, st); }
