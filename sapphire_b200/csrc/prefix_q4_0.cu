// prefix_q4_0.cu - a shared prefix over Q4_0 pages (prefix_kernel.cuh).
#include "prefix_kernel.cuh"

cudaError_t prefix_run_q4_0(const PrefixParams &p, cudaStream_t st) { return prefix_launch<DTYPE_Q4_0, false>(p, st); }
