// Attention over int8 caches in float arithmetic: attention_rows_any.cuh.
#include "attention_rows_any.cuh"

int aa_rows_int8(const RowArgs& a, bool float_q, int max_rows, cudaStream_t s) {
    return float_q ? aa_rows<C8_INT8, float>(a, max_rows, s) : aa_rows<C8_INT8, bf16>(a, max_rows, s);
}
int aa_single_int8(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s) {
    return float_q ? aa_single<C8_INT8, float>(a, max_keys, s) : aa_single<C8_INT8, bf16>(a, max_keys, s);
}
