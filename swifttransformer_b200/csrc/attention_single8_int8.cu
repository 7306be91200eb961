// Single tokens over int8 caches: the instances of attention_single8.cuh.
#include "attention_single8.cuh"

int sg_int8(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s) {
    return float_q ? sg_run<C8_INT8, float, true>(a, max_keys, s) : sg_run<C8_INT8, bf16, false>(a, max_keys, s);
}
