// attention_q8_0.cu - the attention kernels of Q8_0 caches.
#include "attention_kernel.cuh"

cudaError_t attn_run_q8_0(const AttnParams &p, cudaStream_t st) { return attn_launch<DTYPE_Q8_0>(p, st); }
