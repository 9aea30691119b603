// attention_q4_0.cu - the attention kernels of Q4_0 caches.
#include "attention_kernel.cuh"

cudaError_t attn_run_q4_0(const AttnParams &p, cudaStream_t st) { return attn_launch<DTYPE_Q4_0>(p, st); }
