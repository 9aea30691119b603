// attention_f32.cu - the attention kernels of F32 caches: rows, queries and
// probabilities in two 11-bit parts each.
#include "attention_kernel.cuh"

cudaError_t attn_run_f32(const AttnParams &p, cudaStream_t st) {
    return attn_wide(p.group) ? attn_launch<DTYPE_F32, true, 2, 2>(p, st) : attn_launch<DTYPE_F32, false, 1, 1>(p, st);
}
