// Attention over bfloat16 and float32 caches, of queries of the same type, in float arithmetic: attention_rows_any.cuh.
#include "attention_rows_any.cuh"

int aa_rows_wide(const RowArgs& a, bool float_q, int max_rows, cudaStream_t s) {
    return float_q ? aa_rows<C8_F32, float>(a, max_rows, s) : aa_rows<C8_BF16, bf16>(a, max_rows, s);
}
int aa_single_wide(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s) {
    return float_q ? aa_single<C8_F32, float>(a, max_keys, s) : aa_single<C8_BF16, bf16>(a, max_keys, s);
}
