// prefix_f32.cu - a shared prefix over F32 pages (prefix_kernel.cuh).
#include "prefix_kernel.cuh"

cudaError_t prefix_run_f32(const PrefixParams &p, cudaStream_t st) { return prefix_launch<DTYPE_F32, false>(p, st); }
