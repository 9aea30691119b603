// prefix_q8_0.cu - a shared prefix over Q8_0 pages (prefix_kernel.cuh).
#include "prefix_kernel.cuh"

cudaError_t prefix_run_q8_0(const PrefixParams &p, cudaStream_t st) { return prefix_launch<DTYPE_Q8_0, false>(p, st); }
