// Single tokens over e4m3 caches: the instances of attention_single8.cuh.
#include "attention_single8.cuh"

int sg_e4m3(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s) {
    return float_q ? sg_run<C8_E4M3, float, true>(a, max_keys, s) : sg_run<C8_E4M3, bf16, false>(a, max_keys, s);
}
