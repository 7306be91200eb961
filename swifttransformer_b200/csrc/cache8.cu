// Split a fused q|k|v projection, add its bias, keep q, and quantise k and v into the paged 8-bit cache (cache8.cuh) as they are
// written; and rows of that cache read back.  The 16- and 32-bit counterpart is kv_cache.cu; the reference keeps its cache in
// the type of its activations (src/csrc/kernel/kvcache_mgmt.cu:29-80).
//
// A row of head_dim elements is held by a group of 1 to 32 lanes, eight elements each, from the load to the store: the bias sum,
// the largest magnitude (butterflies inside the group), the codes.  So a row is read once and written once, which is the floor;
// a decode step's write is bound by the launch and the chain position, request -> slot -> page, which runs beside the loads (8 tokens
// with their rows read back: 5.5 us), a prompt's by the loads that its blocks have under way (2000 tokens of 32 heads of 128: 25 us,
// 3.3 TB/s; fewer instructions, of 150 for eight elements of a warp, and a shorter chain changed nothing).
//
// Rounding: t = x * (1 / scale) is off by less than 2^-22 of itself.  Where no t of a thread's eight is that near the middle between two
// codes, their roundings are those of the exact quotients; otherwise (of eight numbers spread over the codes one time in a thousand
// for int8, in eight thousand for e4m3; zeros never) the quotients are formed in 64 bits, whose rounding can neither reach nor leave a
// middle: a quotient of two 24-bit numbers that is not such a middle, of at most 9 bits, is further than 2^-34 of itself away from
// it.  The scale likewise: max|x| (1 / M) in 64 bits, rounded once.
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
template <int FORM> __device__ __forceinline__ uint2 c8_codes(const float* x, float scale) {
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(inv) : "f"(scale));     // 1 ulp; 2^-126 <= scale < 2^122: neither end is subnormal
    uint32_t w[2];
    bool near;
    if (FORM == C8_INT8) {
        // t + 1.5 2^23 has round(t) in its low byte
        constexpr float MAGIC = 12582912.f;
        uint32_t u[8];
        float off = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float t = x[i] * inv, m = t + MAGIC;
            u[i] = __float_as_uint(m);
            off = fmaxf(off, fabsf(t - (m - MAGIC)));
        }
        near = off > 0.5f - 0x1p-14f;                                  // |t| <= 127 (1 + 2^-22): off by 2^-15 at most
#pragma unroll
        for (int k = 0; k < 2; ++k)
            w[k] = __byte_perm(__byte_perm(u[4 * k], u[4 * k + 1], 0x0040), __byte_perm(u[4 * k + 2], u[4 * k + 3], 0x0040), 0x5410);
    } else {
        // the middle between two codes from 2^-6 on: the bits behind the third are 1000...
        uint32_t least = 0xffffffffu, small = 0xffffffffu;             // small: twice the bits of the least magnitude but zero, less one
        uint32_t h[4];
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            t[i] = x[i] * inv;
            least = min(least, (__float_as_uint(t[i]) + (8u - 0x80000u)) & 0xfffffu);
            small = min(small, 2u * __float_as_uint(t[i]) - 1u);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = c8_two_e4m3(t[2 * i], t[2 * i + 1]);
        near = least < 16u;
        if (small < 2u * 0x3c800000u - 1u) {
            // below 2^-6, where the codes are multiples of 2^-9 (t off by less than 2^-28: 2^-19 of these)
            constexpr float MAGIC = 12582912.f;
            float off = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = t[i] * 512.f;
                off = fmaxf(off, fabsf(t[i]) < 0x1p-6f ? fabsf(u - ((u + MAGIC) - MAGIC)) : 0.f);
            }
            near |= off > 0.5f - 0x1p-17f;
        }
        w[0] = h[0] | h[1] << 16;
        w[1] = h[2] | h[3] << 16;
    }
    if (near) {
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            uint32_t v = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) v |= c8_exact<FORM>(k ? x[4 + i] : x[i], scale) << (8 * i);
            w[k] = v;
        }
    }
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ float c8_max_nan(float a, float b) {       // of magnitudes; NaN if one is
    float d;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}
// the scale of a row whose largest magnitude this is (or NaN), and whether the row is finite
template <int FORM> __device__ __forceinline__ float c8_scale(float amax, bool& finite) {
    finite = amax < INFINITY;
    if (!finite) return __uint_as_float(0x7fffffffu);
    return fmaxf(__double2float_rn((double)amax * (FORM == C8_INT8 ? 1.0 / 127.0 : 1.0 / 448.0)), C8_TINY);
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

// eight elements as they lie in memory, and as floats
template <typename T> struct Eight;
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = load4(p); b = load4(p + 4); }
    __device__ __forceinline__ void clear() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void floats(float* f) const {
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
};
template <> struct Eight<bf16> {
    uint4 u;
    __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void clear() { u = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void floats(float* f) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};
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

// G lanes per row of d <= 8 G elements (d a multiple of 8), TURN rows per thread, all loaded before the first is worked on and kept as
// they were loaded.
template <typename T, int FORM, int G, int TURN, bool FULL>
__global__ void __launch_bounds__(C8_THREADS, 6) cache8_write_kernel(const Cache8Write a) {
    const int t = blockIdx.x;
    const int pos = __ldg(a.positions + t), seq = __ldg(a.seq_of_token + t);       // (a padding token's request may be any number)
    constexpr int PER = C8_THREADS / G;                  // rows of a turn
    const int nkv = a.kv.nkv, d = FULL ? 8 * G : a.d, rows = a.nh + 2 * nkv;       // FULL: every lane of a group has eight elements
    const int lane = threadIdx.x % G, e = 8 * lane;
    const int first = blockIdx.y * (PER * TURN) + threadIdx.x / G;
    const bool in = FULL || e < d;
    const size_t at = ((size_t)t * rows + first) * d + e;
    const T* src = (const T*)a.qkv + at;
    Eight<T> held[TURN];
#pragma unroll
    for (int j = 0; j < TURN; ++j) {
        const int r = first + j * PER;
        held[j].clear();
        if (in && r < rows && (r >= a.nh || a.q_out)) held[j].load(src + (size_t)(j * PER) * d);
    }
    int page = -1;
    uint32_t row0 = 0;                                   // of key head 0; a page holds all heads' keys, then all heads' values
    if (a.write_kv && pos >= 0) {        // pos < 0: a padding token, nothing is cached
        page = a.kv.page(a.kv.table + (size_t)__ldg(a.slots + seq) * a.kv.max_pages, pos);
        row0 = a.kv.row0(page, 0, 0) + a.kv.offset(pos, a.kv.page_index(pos));
        if (page < 0 && threadIdx.x == 0) atomicExch(a.kv.status, 1);
    }
#pragma unroll
    for (int j = 0; j < TURN; ++j) {
        const int r = first + j * PER;                   // the same for the lanes of a group; a group stays together below
        const bool live = r < rows && in, query = r < a.nh;
        float f[8];
        held[j].floats(f);
        if (live && a.bias) {
            const float* bias = a.bias + (first + j * PER) * d + e;
            const float4 b0 = load4(bias), b1 = load4(bias + 4);
            f[0] += b0.x; f[1] += b0.y; f[2] += b0.z; f[3] += b0.w;
            f[4] += b1.x; f[5] += b1.y; f[6] += b1.z; f[7] += b1.w;
        }
        float amax = 0.f;
        if (!__all_sync(0xffffffffu, query)) {
            amax = c8_max_nan(c8_max_nan(c8_max_nan(f[0], f[1]), c8_max_nan(f[2], f[3])), c8_max_nan(c8_max_nan(f[4], f[5]), c8_max_nan(f[6], f[7])));
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) amax = c8_max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        }
        if (!live) continue;
        if (query) {
            if (a.q_out) c8_store8((T*)a.q_out + ((size_t)t * a.nh + r) * d + e, f);
        } else if (page >= 0) {
            bool finite;
            const float scale = c8_scale<FORM>(amax, finite);
            const uint32_t row = row0 + (uint32_t)(r - a.nh) * a.kv.page_size;
            const uint2 c = finite ? c8_codes<FORM>(f, scale) : make_uint2(0u, 0u);
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
        float amax = 0.f;
        for (int e = lane; e < d; e += 32) amax = c8_max_nan(amax, to_f32(src[e]) + (bias ? bias[e] : 0.f));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = c8_max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
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
    // Two rows per thread once that still leaves two blocks for every SM, else one, so that a decode step's rows are spread over more
    // SMs.  (A block's life is the chain of loads to its page: 2000 tokens of 32 heads of 128 take 25 us with two rows and six
    // blocks on an SM, 28 with four rows, whose registers leave four blocks.)
    const int by2 = (rows + 2 * per - 1) / (2 * per);
    const dim3 grid2(n, by2), grid1(n, (rows + per - 1) / per);
    if ((long long)by2 * n >= 2 * st_sm_count()) {
        if (a.d == 8 * G) cache8_write_kernel<T, FORM, G, 2, true><<<grid2, C8_THREADS, 0, s>>>(a);
        else cache8_write_kernel<T, FORM, G, 2, false><<<grid2, C8_THREADS, 0, s>>>(a);
    } else {
        if (a.d == 8 * G) cache8_write_kernel<T, FORM, G, 1, true><<<grid1, C8_THREADS, 0, s>>>(a);
        else cache8_write_kernel<T, FORM, G, 1, false><<<grid1, C8_THREADS, 0, s>>>(a);
    }
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

// what both entry points take, as the caller lays it out; act: 0 float, 1 bfloat16; form: C8_INT8 or C8_E4M3; d up to 256
struct Cache8Call {
    const void* qkv;
    const float* bias;
    void* q_out;
    void* pool;
    float* scales;
    const int* positions;
    const int* seq_of_token;
    const int* slots;
    const int* block_table;
    int* status;
    void* out;                      // rows read back
    int max_pages, num_pages, n_layers, layer, n_tokens, nh, nkv, d, page_size, write_kv, act, form;
};
static_assert(sizeof(Cache8Call) == 11 * 8 + 12 * 4, "the caller lays this out field by field");

static int c8_check(const Cache8Call& c) {
    if (c.nkv <= 0 || c.d <= 0 || c.page_size <= 0 || c.layer < 0 || c.layer >= c.n_layers || c.max_pages <= 0 || c.num_pages <= 0 || !c.status)
        return ST_ERR_BAD_ARG;
    if (c.d > 256 || c.nkv > (1 << 15) || !c8_rows_fit(c.num_pages, c.n_layers, c.nkv, c.page_size)) return ST_ERR_TOO_LARGE;
    return 0;
}
static PagedKV c8_kv(const Cache8Call& c) {
    return PagedKV{(const unsigned char*)c.pool, c.scales, c.block_table, c.max_pages, c.num_pages, c.n_layers, c.layer, c.nkv, c.page_size,
                   c8_shift(c.page_size), c8_reach(c.max_pages, c.page_size), c.status};
}
ST_EXPORT int st_qkv_to_cache8(const Cache8Call* c, void* stream) {
    if (c->n_tokens <= 0) return 0;
    const int bad = c8_check(*c);
    if (bad) return bad;
    if (c->nh <= 0) return ST_ERR_BAD_ARG;
    if ((long long)c->nh + 2ll * c->nkv > (1 << 16)) return ST_ERR_TOO_LARGE;
    const Cache8Write a{c->qkv, c->bias, c->q_out, (unsigned char*)c->pool, c->scales, c->positions, c->seq_of_token, c->slots, c8_kv(*c),
                        c->nh, c->d, c->write_kv};
    const int act = c->act, form = c->form, n_tokens = c->n_tokens;
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
    const int t = blockIdx.x, pos = __ldg(positions + t), seq = __ldg(seq_of_token + t);
    if (pos < 0) return;
    const int page = kv.page(kv.table + (size_t)__ldg(slots + seq) * kv.max_pages, pos);
    const uint32_t row0 = page >= 0 ? kv.row0(page, 0, 0) + kv.offset(pos, kv.page_index(pos)) : 0u;    // all heads' keys, then all values
    if (page < 0 && threadIdx.x == 0 && kv.status) atomicExch(kv.status, 1);
    const int per = d / W, total = 2 * kv.nkv * per;
    T* dst = out + (size_t)t * 2 * kv.nkv * d;
#pragma unroll 4
    for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < total; i += gridDim.y * blockDim.x) {
        const int r = i / per, e = (i - r * per) * W;
        float f[W];
#pragma unroll
        for (int k = 0; k < W; ++k) f[k] = 0.f;
        if (page >= 0) {
            const uint32_t row = row0 + (uint32_t)r * kv.page_size;
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
    if (y > 65535) y = 65535;
    if (vec) cache8_rows_kernel<T, FORM, 8><<<dim3(n, y), C8_THREADS, 0, s>>>(kv, (T*)out, positions, seq_of_token, slots, d);
    else cache8_rows_kernel<T, FORM, 1><<<dim3(n, y), C8_THREADS, 0, s>>>(kv, (T*)out, positions, seq_of_token, slots, d);
    return st_launch_status();
}

ST_EXPORT int st_cache8_rows(const Cache8Call* c, void* stream) {
    if (c->n_tokens <= 0) return 0;
    const int bad = c8_check(*c);
    if (bad) return bad;
    const PagedKV kv = c8_kv(*c);
    void* out = c->out;
    const int *positions = c->positions, *seq_of_token = c->seq_of_token, *slots = c->slots;
    const int act = c->act, form = c->form, n_tokens = c->n_tokens, d = c->d;
    cudaStream_t s = (cudaStream_t)stream;
    if (act == 0 && form == C8_INT8) return c8_launch_rows<float, C8_INT8>(kv, out, positions, seq_of_token, slots, n_tokens, d, s);
    if (act == 0 && form == C8_E4M3) return c8_launch_rows<float, C8_E4M3>(kv, out, positions, seq_of_token, slots, n_tokens, d, s);
    if (act == 1 && form == C8_INT8) return c8_launch_rows<bf16, C8_INT8>(kv, out, positions, seq_of_token, slots, n_tokens, d, s);
    if (act == 1 && form == C8_E4M3) return c8_launch_rows<bf16, C8_E4M3>(kv, out, positions, seq_of_token, slots, n_tokens, d, s);
    return ST_ERR_BAD_DTYPE;
}
