// The forms a paged cache may have, and where its rows lie.
//
// An 8-bit cache is a pair of tensors
//   pool  [page][layer][K|V][kv_head][position in page][head_dim]   one byte per element: int8 or e4m3
//   scales[page][layer][K|V][kv_head][position in page]             float
// an element's value is its code's value times its row's scale.  The scale of a row x is max(max|x| / M, 2^-126) in float with
// M = 127 (int8) or 448 (e4m3), its codes are x / scale rounded to the nearest number the form has, ties to even, by the exact
// quotient.  A row with a NaN or an infinity has the scale NaN and codes 0: whoever sees the row reads NaN, and whoever has it
// masked multiplies finite codes.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

#define C8_INT8 0
#define C8_E4M3 1
#define C8_BF16 2
#define C8_F32 3

#define C8_TINY 1.17549435e-38f          // 2^-126: the least scale

__host__ __device__ constexpr int c8_bytes(int form) { return form == C8_F32 ? 4 : form == C8_BF16 ? 2 : 1; }

// A paged cache as the kernels see it.
struct PagedKV {
    const unsigned char* pool;
    const float* scales;                 // null for 16- and 32-bit caches
    const int* table;                    // [slots][max_pages]
    int max_pages, num_pages, n_layers, layer, nkv, page_size, page_shift;   // page_shift: log2 of page_size, or -1
    int reach;                           // positions that the table has room for
    int* status;                         // set to 1 where a needed key has no page

    __device__ __forceinline__ int page_index(int key) const { return page_shift >= 0 ? key >> page_shift : key / page_size; }
    // the page of `key` in a request's row of the table, or -1
    __device__ __forceinline__ int page(const int* row, int key) const {
        const int j = page_index(key);
        if (j >= max_pages) return -1;
        const int p = __ldg(row + j);
        return (unsigned)p < (unsigned)num_pages ? p : -1;
    }
    // the pool's row of position 0 of a page, for keys (0) or values (1) of a head: below 2^32, the launchers see to it
    __device__ __forceinline__ uint32_t row0(int page, int which, int head) const {
        return ((((uint32_t)page * n_layers + layer) * 2 + which) * nkv + head) * (uint32_t)page_size;
    }
    __device__ __forceinline__ int offset(int key, int index) const { return key - index * page_size; }
};

static inline int c8_shift(int page_size) {
    for (int s = 0; s < 30; ++s)
        if ((1 << s) == page_size) return s;
    return -1;
}
// a little below 2^31 at most: sums of a position and a run's keys stay in an int
static inline int c8_reach(int max_pages, int page_size) {
    const long long n = (long long)max_pages * page_size;
    return n < 0x7fff0000ll ? (int)n : 0x7fff0000;
}
// rows of a pool fit 32-bit unsigned indices
static inline bool c8_rows_fit(long long num_pages, int n_layers, int nkv, int page_size) {
    return num_pages * n_layers * 2 * nkv * page_size < (1ll << 32);
}

// one element as a float (without its row's scale)
template <int FORM> __device__ __forceinline__ float c8_value(const unsigned char* pool, size_t i) {
    if (FORM == C8_INT8) return (float)reinterpret_cast<const signed char*>(pool)[i];
    if (FORM == C8_E4M3) {
        const __half_raw h = __nv_cvt_fp8_to_halfraw(pool[i], __NV_E4M3);
        return __half2float(*reinterpret_cast<const __half*>(&h));
    }
    if (FORM == C8_BF16) return __bfloat162float(reinterpret_cast<const bf16*>(pool)[i]);
    return reinterpret_cast<const float*>(pool)[i];
}

// ---- codes as pairs of halves, exactly: int8 and e4m3 numbers are 16-bit floats ------------------------------------
__device__ __forceinline__ uint32_t c8_hsub2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ void c8_e4m3x4(uint32_t w, uint32_t& lo, uint32_t& hi) {       // the low two bytes, the high two
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}\n"
        : "=r"(lo), "=r"(hi) : "r"(w));
}
// int8: the byte c + 128 behind the exponent of 1024 is the half 1024 + 128 + c; 1152 less is c
#define C8_BIAS 0x64806480u               // (half 1152) twice, which is also 0x6400 with the sign bit of the byte flipped
// four codes of one word -> (c0, c1), (c2, c3)
template <int FORM> __device__ __forceinline__ void c8_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (FORM == C8_INT8) {
        const uint32_t u = w ^ 0x80808080u;
        lo = c8_hsub2(__byte_perm(u, 0x64646464u, 0x4140), C8_BIAS);
        hi = c8_hsub2(__byte_perm(u, 0x64646464u, 0x4342), C8_BIAS);
    } else {
        c8_e4m3x4(w, lo, hi);
    }
}
__device__ __forceinline__ uint32_t c8_biased(uint32_t bytes) {      // bytes 0 and 2 behind the exponent of 1024, sign bits flipped
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;\n" : "=r"(d) : "r"(bytes), "r"(0x00ff00ffu), "r"(C8_BIAS));      // (bytes & mask) ^ bias in one
    return d;
}
// words a and b of two rows -> the pairs (a_i, b_i), i = 0..3
template <int FORM> __device__ __forceinline__ void c8_pairs(uint32_t a, uint32_t b, uint32_t* out) {
    if (FORM == C8_INT8) {
        out[0] = c8_hsub2(c8_biased(__byte_perm(a, b, 0x0400)), C8_BIAS);
        out[1] = c8_hsub2(c8_biased(__byte_perm(a, b, 0x0501)), C8_BIAS);
        out[2] = c8_hsub2(c8_biased(__byte_perm(a, b, 0x0602)), C8_BIAS);
        out[3] = c8_hsub2(c8_biased(__byte_perm(a, b, 0x0703)), C8_BIAS);
    } else {
        c8_e4m3x4(__byte_perm(a, b, 0x5140), out[0], out[1]);
        c8_e4m3x4(__byte_perm(a, b, 0x7362), out[2], out[3]);
    }
}
