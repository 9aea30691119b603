// attention_bf16.cu - the attention kernels of BF16 caches.  bf16 queries are one
// part and probabilities two (2^-18 against the output's 2^-9); fp32 and fp16
// ones take three.
#include "attention_kernel.cuh"

cudaError_t attn_run_bf16(const AttnParams &p, cudaStream_t st) {
    if (p.io == DTYPE_BF16)
        return attn_wide(p.group) ? attn_launch<DTYPE_BF16, true, 1, 2>(p, st) : attn_launch<DTYPE_BF16, false, 1, 1>(p, st);
    return attn_wide(p.group) ? attn_launch<DTYPE_BF16, true, 3, 3>(p, st) : attn_launch<DTYPE_BF16, false, 2, 2>(p, st);
}
