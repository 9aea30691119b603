// prefix_bf16.cu - a shared prefix over BF16 pages (prefix_kernel.cuh).
#include "prefix_kernel.cuh"

// Under bf16 queries the rows are operands as they are.
cudaError_t prefix_run_bf16(const PrefixParams &p, cudaStream_t st) {
    return p.io == DTYPE_BF16 ? prefix_launch<DTYPE_BF16, true>(p, st) : prefix_launch<DTYPE_BF16, false>(p, st);
}
