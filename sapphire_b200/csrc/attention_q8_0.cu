// attention_q8_0.cu - the attention kernels of Q8_0 caches.  Two fp16 parts hold
// 24 bits; a bf16 query is one exactly, and one of the probability (2^-12) is
// enough under a bf16 output.
#include "attention_kernel.cuh"

cudaError_t attn_run_q8_0(const AttnParams &p, cudaStream_t st) {
    if (!attn_wide(p.group)) return attn_launch<DTYPE_Q8_0, false, 1, 1>(p, st);
    return p.io == DTYPE_BF16 ? attn_launch<DTYPE_Q8_0, true, 1, 1>(p, st) : attn_launch<DTYPE_Q8_0, true, 2, 2>(p, st);
}
