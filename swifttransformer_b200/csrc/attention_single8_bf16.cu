// Single tokens over bfloat16 caches, behind a shared prefix: the instances of attention_single8.cuh.
#include "attention_single8.cuh"

int sg_bf16(const SingleArgs& a, int max_keys, cudaStream_t s) {
    // a weight in one bfloat16 number would be the largest error; the other four columns have room for the second
    return a.group <= 4 ? sg_run<C8_BF16, bf16, true>(a, max_keys, s) : sg_run<C8_BF16, bf16, false>(a, max_keys, s);
}
