// attention_f32.cu - the attention kernels of F32 caches.
#include "attention_kernel.cuh"

cudaError_t attn_run_f32(const AttnParams &p, cudaStream_t st) { return attn_launch<DTYPE_F32>(p, st); }
