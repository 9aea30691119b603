// attention_f16.cu - the attention kernels of F16 caches.
#include "attention_kernel.cuh"

cudaError_t attn_run_f16(const AttnParams &p, cudaStream_t st) { return attn_launch<DTYPE_F16>(p, st); }
