// Single tokens over bfloat16 caches, behind a shared prefix: the instances of attention_single8.cuh.
#include "attention_single8.cuh"

int sg_bf16(const SingleArgs& a, int max_keys, cudaStream_t s) { return sg_run<C8_BF16, bf16>(a, max_keys, s); }
