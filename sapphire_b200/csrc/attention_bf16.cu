// attention_bf16.cu - the attention kernels of BF16 caches.
#include "attention_kernel.cuh"

cudaError_t attn_run_bf16(const AttnParams &p, cudaStream_t st) { return attn_launch<DTYPE_BF16>(p, st); }
