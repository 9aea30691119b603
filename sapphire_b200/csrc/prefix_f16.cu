// prefix_f16.cu - a shared prefix over F16 pages (prefix_kernel.cuh).
#include "prefix_kernel.cuh"

cudaError_t prefix_run_f16(const PrefixParams &p, cudaStream_t st) { return prefix_launch<DTYPE_F16, false>(p, st); }
