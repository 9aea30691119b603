// attention_f16.cu - the attention kernels of F16 caches.  Two fp16 parts hold
// 24 bits; a bf16 query is one exactly, and one of the probability (2^-12) is
// enough under a bf16 output.
#include "attention_kernel.cuh"

cudaError_t attn_run_f16(const AttnParams &p, cudaStream_t st) {
    if (!attn_wide(p.group)) return attn_launch<DTYPE_F16, false, 1, 1>(p, st);
    return p.io == DTYPE_BF16 ? attn_launch<DTYPE_F16, true, 1, 1>(p, st) : attn_launch<DTYPE_F16, true, 2, 2>(p, st);
}
