// Split a fused q|k|v projection, add its bias, keep q, and quantise k and v into the paged 8-bit cache (cache8.cuh) as they are
// written; and rows of that cache read back.  The 16- and 32-bit counterpart is kv_cache.cu; the reference keeps its cache in
// the type of its activations (src/csrc/kernel/kvcache_mgmt.cu:29-80).
//
// A row of head_dim elements is held by a group of 1 to 32 lanes, eight elements each, from the load to the store: the bias sum,
// the largest magnitude (butterflies inside the group), the codes.  So a row is read once and written once, which is the floor;
// the write of 2000 tokens of OPT-6.7B (32 heads of 128) is bound by memory, a decode step's by the launch and the chain
// position -> request -> slot -> page, which runs beside the loads.
//
// Rounding: t = x * (1 / scale) is off by less than 2^-22 of itself, so t (1 - 2^-21) and t (1 + 2^-21) bracket the exact quotient;
// where both round to the same code that is the code.  Otherwise (about one in ten thousand) the quotient is formed in 64 bits,
// whose rounding can neither reach nor leave the middle between two codes: a quotient of two 24-bit numbers that is not such
// a middle, of at most 9 bits, is further than 2^-34 of itself away from it.
#include "cache8.cuh"

#define C8_THREADS 256

__device__ __forceinline__ uint32_t c8_two_e4m3(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
template <int FORM> __device__ __noinline__ uint32_t c8_exact(float x, float scale) {
    const double t = (double)x / (double)scale;
    if (FORM == C8_INT8) return (uint32_t)(int)fmin(fmax(rint(t), -127.0), 127.0) & 0xffu;
    // to float by cutting, the last bit set where something was cut: the rounding to e4m3 that follows is then exact
    float f = __double2float_rz(t);
    if ((double)f != t) f = __uint_as_float(__float_as_uint(f) | 1u);
    return c8_two_e4m3(f, f) & 0xffu;
}
// codes of eight elements, four to a word
template <int FORM> __device__ __forceinline__ uint2 c8_codes(const float* x, float scale, float inv) {
    uint32_t w[2] = {0, 0};
    constexpr float DN = 1.f - 0x1p-21f, UP = 1.f + 0x1p-21f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float t0 = x[i] * inv, t1 = x[i + 1] * inv;
        uint32_t lo, hi;
        if (FORM == C8_INT8) {
            const int a0 = __float2int_rn(t0 * DN), b0 = __float2int_rn(t0 * UP), a1 = __float2int_rn(t1 * DN), b1 = __float2int_rn(t1 * UP);
            lo = (a0 & 0xff) | (a1 & 0xff) << 8;
            hi = (b0 & 0xff) | (b1 & 0xff) << 8;
            // t can lie a little above 127: 127 (1 + 2^-21) rounds to 127, no clamp is needed
        } else {
            lo = c8_two_e4m3(t0 * DN, t1 * DN);
            hi = c8_two_e4m3(t0 * UP, t1 * UP);
        }
        if (lo != hi) lo = c8_exact<FORM>(x[i], scale) | c8_exact<FORM>(x[i + 1], scale) << 8;
        w[i >> 2] |= (lo & 0xffffu) << ((i & 2) * 8);
    }
    return make_uint2(w[0], w[1]);
}
// the scale of a row whose largest magnitude has these bits, and whether the row is finite
template <int FORM> __device__ __forceinline__ float c8_scale(uint32_t amax_bits, bool& finite) {
    finite = amax_bits < 0x7f800000u;
    if (!finite) return __uint_as_float(0x7fffffffu);
    return fmaxf(__fdiv_rn(__uint_as_float(amax_bits), FORM == C8_INT8 ? 127.f : 448.f), C8_TINY);
}

struct Cache8Write {
    const void* qkv;
    const float* bias;
    void* q_out;
    unsigned char* pool;
    float* scales;
    const int* positions;
    const int* seq_of_token;
    const int* slots;
    PagedKV kv;
    int nh, d, write_kv;
};

template <typename T> __device__ __forceinline__ void c8_load8(const T* p, float* f);
template <> __device__ __forceinline__ void c8_load8<float>(const float* p, float* f) {
    const float4 a = load4(p), b = load4(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
template <> __device__ __forceinline__ void c8_load8<bf16>(const bf16* p, float* f) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void c8_store8(float* p, const float* f) {
    store4(p, make_float4(f[0], f[1], f[2], f[3]));
    store4(p + 4, make_float4(f[4], f[5], f[6], f[7]));
}
__device__ __forceinline__ void c8_store8(bf16* p, const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// G lanes per row of d <= 8 G elements (d a multiple of 8), TURN rows per thread, all loaded before the first is worked on
template <typename T, int FORM, int G, int TURN>
__global__ void __launch_bounds__(C8_THREADS) cache8_write_kernel(const Cache8Write a) {
    const int t = blockIdx.x;
    const int nkv = a.kv.nkv, d = a.d, rows = a.nh + 2 * nkv;
    const int lane = threadIdx.x % G, e = 8 * lane;
    const int first = blockIdx.y * (C8_THREADS / G * TURN) + threadIdx.x / G;
    const T* src = (const T*)a.qkv + (size_t)t * rows * d + e;
    const bool in = e < d;
    float f[TURN][8];
#pragma unroll
    for (int j = 0; j < TURN; ++j) {
        const int r = first + j * (C8_THREADS / G);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] = 0.f;
        if (in && r < rows && (r >= a.nh || a.q_out)) c8_load8<T>(src + (size_t)r * d, f[j]);
    }
    const int pos = a.positions[t];
    int page = -1, off = 0;
    if (a.write_kv && pos >= 0) {        // pos < 0: a padding token, nothing is cached
        const int index = a.kv.page_index(pos);
        page = a.kv.page(a.kv.table + (size_t)a.slots[a.seq_of_token[t]] * a.kv.max_pages, pos);
        off = a.kv.offset(pos, index);
        if (page < 0 && threadIdx.x == 0) atomicExch(a.kv.status, 1);
    }
#pragma unroll
    for (int j = 0; j < TURN; ++j) {
        const int r = first + j * (C8_THREADS / G);      // the same for the lanes of a group; a group stays together below
        const bool live = r < rows && in;
        if (live && a.bias) {
            const float4 b0 = load4(a.bias + (size_t)r * d + e), b1 = load4(a.bias + (size_t)r * d + e + 4);
            f[j][0] += b0.x; f[j][1] += b0.y; f[j][2] += b0.z; f[j][3] += b0.w;
            f[j][4] += b1.x; f[j][5] += b1.y; f[j][6] += b1.z; f[j][7] += b1.w;
        }
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(f[j][i]) & 0x7fffffffu);
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (!live) continue;
        if (r < a.nh) {
            if (a.q_out) c8_store8((T*)a.q_out + ((size_t)t * a.nh + r) * d + e, f[j]);
        } else if (page >= 0) {
            const int which = r - a.nh >= nkv, head = r - a.nh - which * nkv;
            bool finite;
            const float scale = c8_scale<FORM>(amax, finite);
            const uint32_t row = a.kv.row0(page, which, head) + off;
            const uint2 c = finite ? c8_codes<FORM>(f[j], scale, __frcp_rn(scale)) : make_uint2(0u, 0u);
            *reinterpret_cast<uint2*>(a.pool + (size_t)row * d + e) = c;
            if (lane == 0) a.scales[row] = scale;
        }
    }
}

// any head size and alignment: a warp per row, element by element
template <typename T, int FORM>
__global__ void __launch_bounds__(C8_THREADS) cache8_write_any_kernel(const Cache8Write a) {
    const int t = blockIdx.x, nkv = a.kv.nkv, d = a.d, rows = a.nh + 2 * nkv, lane = threadIdx.x & 31;
    const int pos = a.positions[t];
    int page = -1, off = 0;
    if (a.write_kv && pos >= 0) {
        page = a.kv.page(a.kv.table + (size_t)a.slots[a.seq_of_token[t]] * a.kv.max_pages, pos);
        off = a.kv.offset(pos, a.kv.page_index(pos));
        if (page < 0 && threadIdx.x == 0) atomicExch(a.kv.status, 1);
    }
    for (int r = blockIdx.y * (C8_THREADS / 32) + (threadIdx.x >> 5); r < rows; r += gridDim.y * (C8_THREADS / 32)) {
        const T* src = (const T*)a.qkv + ((size_t)t * rows + r) * d;
        const float* bias = a.bias ? a.bias + (size_t)r * d : nullptr;
        if (r < a.nh) {
            if (a.q_out)
                for (int e = lane; e < d; e += 32)
                    ((T*)a.q_out)[((size_t)t * a.nh + r) * d + e] = from_f32<T>(to_f32(src[e]) + (bias ? bias[e] : 0.f));
            continue;
        }
        if (page < 0) continue;
        uint32_t amax = 0;
        for (int e = lane; e < d; e += 32)
            amax = max(amax, __float_as_uint(to_f32(src[e]) + (bias ? bias[e] : 0.f)) & 0x7fffffffu);
        amax = __reduce_max_sync(0xffffffffu, amax);
        const int which = r - a.nh >= nkv, head = r - a.nh - which * nkv;
        bool finite;
        const float scale = c8_scale<FORM>(amax, finite);
        const uint32_t row = a.kv.row0(page, which, head) + off;
        for (int e = lane; e < d; e += 32)
            a.pool[(size_t)row * d + e] = finite ? (unsigned char)c8_exact<FORM>(to_f32(src[e]) + (bias ? bias[e] : 0.f), scale) : 0;
        if (lane == 0) a.scales[row] = scale;
    }
}

template <typename T, int FORM, int G>
static int c8_launch_write(const Cache8Write& a, int n, cudaStream_t s) {
    const int rows = a.nh + 2 * a.kv.nkv, per = C8_THREADS / G;
    // Four rows per thread once that still leaves two blocks for every SM, else one: with four, their loads are under way together;
    // with one, a decode step's rows are spread over more SMs.
    const int by4 = (rows + 4 * per - 1) / (4 * per);
    if ((long long)by4 * n >= 2 * st_sm_count())
        cache8_write_kernel<T, FORM, G, 4><<<dim3(n, by4), C8_THREADS, 0, s>>>(a);
    else
        cache8_write_kernel<T, FORM, G, 1><<<dim3(n, (rows + per - 1) / per), C8_THREADS, 0, s>>>(a);
    return st_launch_status();
}
template <typename T, int FORM> static int c8_launch_write(const Cache8Write& a, int n, cudaStream_t s) {
    const bool vec = a.d % 8 == 0 && aligned16(a.qkv) && aligned16(a.bias) && aligned16(a.q_out) && aligned16(a.pool);
    if (!vec) {
        const int rows = a.nh + 2 * a.kv.nkv, per = C8_THREADS / 32, y = (rows + per - 1) / per;
        cache8_write_any_kernel<T, FORM><<<dim3(n, y < 65535 ? y : 65535), C8_THREADS, 0, s>>>(a);
        return st_launch_status();
    }
    if (a.d <= 32) return c8_launch_write<T, FORM, 4>(a, n, s);
    if (a.d <= 64) return c8_launch_write<T, FORM, 8>(a, n, s);
    if (a.d <= 128) return c8_launch_write<T, FORM, 16>(a, n, s);
    return c8_launch_write<T, FORM, 32>(a, n, s);
}

// act: 0 float, 1 bfloat16; form: C8_INT8 or C8_E4M3; d up to 256
ST_EXPORT int st_qkv_to_cache8(const void* qkv, const float* bias, void* q_out, void* pool, float* scales, const int* positions,
                               const int* seq_of_token, const int* slots, const int* block_table, int max_pages, int num_pages,
                               int n_layers, int layer, int n_tokens, int nh, int nkv, int d, int page_size, int write_kv, int* status,
                               int act, int form, void* stream) {
    if (n_tokens <= 0) return 0;
    if (nh <= 0 || nkv <= 0 || d <= 0 || page_size <= 0 || layer < 0 || layer >= n_layers || max_pages <= 0 || num_pages <= 0 || !status)
        return ST_ERR_BAD_ARG;
    if (d > 256) return ST_ERR_TOO_LARGE;
    if (!c8_rows_fit(num_pages, n_layers, nkv, page_size) || (long long)nh + 2ll * nkv > (1 << 16)) return ST_ERR_TOO_LARGE;
    Cache8Write a{qkv, bias, q_out, (unsigned char*)pool, scales, positions, seq_of_token, slots,
                  PagedKV{(const unsigned char*)pool, scales, block_table, max_pages, num_pages, n_layers, layer, nkv, page_size,
                          c8_shift(page_size), status}, nh, d, write_kv};
    cudaStream_t s = (cudaStream_t)stream;
    if (act == 0 && form == C8_INT8) return c8_launch_write<float, C8_INT8>(a, n_tokens, s);
    if (act == 0 && form == C8_E4M3) return c8_launch_write<float, C8_E4M3>(a, n_tokens, s);
    if (act == 1 && form == C8_INT8) return c8_launch_write<bf16, C8_INT8>(a, n_tokens, s);
    if (act == 1 && form == C8_E4M3) return c8_launch_write<bf16, C8_E4M3>(a, n_tokens, s);
    return ST_ERR_BAD_DTYPE;
}

// ---- rows read back -----------------------------------------------------------------------------------------------
// out[t] = (keys of all heads | values of all heads) of position positions[t] of request seq_of_token[t].  W: elements a thread
// moves at a time (8 or 1).  A token without a page gives zeros and sets the status.
template <typename T, int FORM, int W>
__global__ void __launch_bounds__(C8_THREADS)
cache8_rows_kernel(const PagedKV kv, T* __restrict__ out, const int* __restrict__ positions, const int* __restrict__ seq_of_token,
                   const int* __restrict__ slots, int d) {
    const int t = blockIdx.x, pos = positions[t];
    if (pos < 0) return;
    const int page = kv.page(kv.table + (size_t)slots[seq_of_token[t]] * kv.max_pages, pos);
    const int off = kv.offset(pos, kv.page_index(pos));
    if (page < 0 && threadIdx.x == 0 && kv.status) atomicExch(kv.status, 1);
    const int per = d / W, total = 2 * kv.nkv * per;
    T* dst = out + (size_t)t * 2 * kv.nkv * d;
    for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < total; i += gridDim.y * blockDim.x) {
        const int r = i / per, e = (i - r * per) * W;
        float f[W];
#pragma unroll
        for (int k = 0; k < W; ++k) f[k] = 0.f;
        if (page >= 0) {
            const int which = r >= kv.nkv;
            const uint32_t row = kv.row0(page, which, r - which * kv.nkv) + off;
            const float s = __ldg(kv.scales + row);
            if constexpr (W == 8) {
                const uint2 c = __ldg(reinterpret_cast<const uint2*>(kv.pool + (size_t)row * d + e));
                uint32_t h[4];
                c8_halves<FORM>(c.x, h[0], h[1]);
                c8_halves<FORM>(c.y, h[2], h[3]);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[k]));
                    f[2 * k] = v.x * s; f[2 * k + 1] = v.y * s;
                }
            } else {
                f[0] = c8_value<FORM>(kv.pool, (size_t)row * d + e) * s;
            }
        }
        if constexpr (W == 8) c8_store8(dst + (size_t)r * d + e, f);
        else dst[(size_t)r * d + e] = from_f32<T>(f[0]);
    }
}

template <typename T, int FORM>
static int c8_launch_rows(const PagedKV& kv, void* out, const int* positions, const int* seq_of_token, const int* slots, int n, int d,
                          cudaStream_t s) {
    const bool vec = d % 8 == 0 && aligned16(out) && aligned16(kv.pool);
    const int total = 2 * kv.nkv * d / (vec ? 8 : 1);
    int y = (total + C8_THREADS - 1) / C8_THREADS;
    if (n >= 2 * st_sm_count() && y > 1) y = (y + 3) / 4;      // four turns a thread where the tokens alone fill the device
    if (vec) cache8_rows_kernel<T, FORM, 8><<<dim3(n, y), C8_THREADS, 0, s>>>(kv, (T*)out, positions, seq_of_token, slots, d);
    else cache8_rows_kernel<T, FORM, 1><<<dim3(n, y), C8_THREADS, 0, s>>>(kv, (T*)out, positions, seq_of_token, slots, d);
    return st_launch_status();
}

ST_EXPORT int st_cache8_rows(const void* pool, const float* scales, void* out, const int* positions, const int* seq_of_token,
                             const int* slots, const int* block_table, int max_pages, int num_pages, int n_layers, int layer, int n_tokens,
                             int nkv, int d, int page_size, int* status, int act, int form, void* stream) {
    if (n_tokens <= 0) return 0;
    if (nkv <= 0 || d <= 0 || page_size <= 0 || layer < 0 || layer >= n_layers || max_pages <= 0 || num_pages <= 0) return ST_ERR_BAD_ARG;
    if (d > 256 || nkv > (1 << 15) || !c8_rows_fit(num_pages, n_layers, nkv, page_size)) return ST_ERR_TOO_LARGE;
    const PagedKV kv{(const unsigned char*)pool, scales, block_table, max_pages, num_pages, n_layers, layer, nkv, page_size,
                     c8_shift(page_size), status};
    cudaStream_t s = (cudaStream_t)stream;
    if (act == 0 && form == C8_INT8) return c8_launch_rows<float, C8_INT8>(kv, out, positions, seq_of_token, slots, n_tokens, d, s);
    if (act == 0 && form == C8_E4M3) return c8_launch_rows<float, C8_E4M3>(kv, out, positions, seq_of_token, slots, n_tokens, d, s);
    if (act == 1 && form == C8_INT8) return c8_launch_rows<bf16, C8_INT8>(kv, out, positions, seq_of_token, slots, n_tokens, d, s);
    if (act == 1 && form == C8_E4M3) return c8_launch_rows<bf16, C8_E4M3>(kv, out, positions, seq_of_token, slots, n_tokens, d, s);
    return ST_ERR_BAD_DTYPE;
}
