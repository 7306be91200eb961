// Attention of single query tokens over paged caches in 8 and 16 bits (and, in 16 bits, of the keys behind a shared prefix): one
// block per (token, key head, up to 8 or 16 of its query heads, share of the keys).
//
// Mathematics: s_j = (q . c_j) ks_j, o = sum_j p_j vs_j c'_j / sum_j p_j with the codes c, c' and the rows' scales ks, vs: the
// scales leave both products, whose operands are then exact in 16 bits: codes of either 8-bit form are halves; a bfloat16 query
// is scaled by a power of two per row, so that its largest element lies in [2^14, 2^15), and is a half unless an element is
// 2^-29 of that or less; a float query is the sum of two halves (22 bits; the rest, 2^-23 of an element, is below what 32-bit
// sums round away).  Products go to mma.sync (m16n8k16: 8 or 16 query rows on the row side, eight keys or eight dimensions on
// the other), sums are float.  The weights are p_j vs_j in a half of 2^-11 (for float queries and bfloat16 caches in two
// numbers, the lower one in the row operand's other eight rows, which costs no instruction).
//
// p_j = 2^(s_j - R): R follows the largest of s_j + log2 vs_j in steps: it moves when that exceeds R + 15, and then to 11 below, so
// that p_j vs_j stays below 2^15 and what is 2^-24 of the largest still has a half's full precision.  Sums of 32 (16) keys are formed
// in fresh accumulators and added to the running ones with a float add each: tensor cores cut what they add to a large sum.
//
// Layout: no shared memory on the way in.  A warp walks every n-th run of KT = 32 keys (16 where rows are longer than 64 bytes).
// Lane (g, t) = (lane / 4, lane % 4) reads of each key row that is its column g of a product a quarter in pieces of 16 bytes
// (the order of the summed dimensions is free, the query's is the same), and of the values of KT/4 neighbouring keys an
// eighth of the row.  Keys are dealt to columns so that the KT/4 keys of lane t's scores are those whose values it reads:
// scores, weights and values meet without an exchange between lanes, and each lane looks up two pages per run.
//
// Bound by memory.  What the loads in flight need is covered by many warps: keys of the next run are asked for as soon as this run's
// products have taken theirs, values likewise.
#pragma once
#include "attention_rows.cuh"

#define SG_MAX_WARPS 16

// what the finished row goes through, for all kernels of single tokens
struct SingleArgs {
    const void* q;
    void* out;
    PagedKV kv;
    const int* items;            // tokens, or null: 0 .. n_items - 1
    const int* positions;
    const int* seq_of_token;
    const int* slots;
    const int* info;             // [n_items][3]: keys shared with others, tile, the token's place in it; null: no prefix
    RowPlan plan;                // of the prefix
    RowParts parts;
    int nh, group, d, n_items, splits, row_blocks;
    float scale_log2;
    int window;
};

__device__ __forceinline__ void sg_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ float sg_remote(const float* local, uint32_t rank) {     // the same place in block `rank` of the cluster
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// The warps' parts of R rows x D, then the cluster's, then the prefix's, to the output.  smem: W x R x (D + 2) floats: (R, l) of each
// warp and row, then O.  `rows` of the R are real; head0 is the first one's query head.
template <typename QT>
__device__ __forceinline__ void sg_finish(const SingleArgs& a, float* smem, int W, int R, int rows, int D, int token, int item,
                                          int head0, int key_head) {
    float* ref = smem;
    float* sum = ref + W * R;
    float* acc = sum + W * R;
    __syncthreads();
    // this block's part, into the first warp's place
    for (int i = threadIdx.x; i < rows * D; i += blockDim.x) {
        const int r = i / D;
        float m = -INFINITY;
        for (int w = 0; w < W; ++w) m = fmaxf(m, ref[w * R + r]);
        float o = 0.f;
        for (int w = 0; w < W; ++w) o += ar_weight(ref[w * R + r], m) * acc[((size_t)w * R + r) * D + (i - r * D)];
        acc[(size_t)r * D + (i - r * D)] = o;          // (warp 0's number at this place was read above, by this thread alone)
    }
    __syncthreads();
    if (threadIdx.x < rows) {
        const int r = threadIdx.x;
        float m = -INFINITY, l = 0.f;
        for (int w = 0; w < W; ++w) m = fmaxf(m, ref[w * R + r]);
        for (int w = 0; w < W; ++w) l += ar_weight(ref[w * R + r], m) * sum[w * R + r];
        ref[r] = m;
        sum[r] = l;
    }
    uint32_t rank = 0;
    if (a.splits > 1) {
        asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
        sg_cluster_sync();
    } else {
        __syncthreads();
    }
    RowTile t{};
    int tile = 0, place = 0;
    if (a.info) {
        ST_PDL_WAIT();                                 // the prefix's parts are complete
        tile = a.info[3 * item + 1];
        place = a.info[3 * item + 2];
        t = ar_tile(a.plan, tile);
    }
    QT* out = (QT*)a.out + ((size_t)token * a.nh + head0) * D;
    for (int i = threadIdx.x + rank * blockDim.x; i < rows * D; i += blockDim.x * a.splits) {
        const int r = i / D;
        float m = -INFINITY, l = 0.f, o = 0.f;
        for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.splits > 1 ? sg_remote(ref + r, s) : ref[r]);
        const int row = place * a.group + (head0 - key_head * a.group) + r;
        if (a.info) ar_each_part(a.plan, t, tile, key_head, [&](int slot) { m = fmaxf(m, __ldcg(a.parts.r + (size_t)slot * AR_ROWS + row)); });
        for (int s = 0; s < a.splits; ++s) {
            const float w = ar_weight(a.splits > 1 ? sg_remote(ref + r, s) : ref[r], m);
            l += w * (a.splits > 1 ? sg_remote(sum + r, s) : sum[r]);
            o += w * (a.splits > 1 ? sg_remote(acc + i, s) : acc[i]);
        }
        if (a.info)
            ar_each_part(a.plan, t, tile, key_head, [&](int slot) {
                const size_t at = (size_t)slot * AR_ROWS + row;
                const float w = ar_weight(__ldcg(a.parts.r + at), m);
                l += w * __ldcg(a.parts.l + at);
                o += w * __ldcg(a.parts.o + at * D + (i - r * D));
            });
        out[i] = from_f32<QT>(l == 0.f ? 0.f : o / l);   // no key at all: zeros
    }
    if (a.splits > 1) sg_cluster_sync();               // nobody leaves while others read here
}

__device__ __forceinline__ void sg_mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1, bool half) {
    if (half)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool HALF> __device__ __forceinline__ uint32_t sg_pack(float a, float b) {
    if (HALF) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool HALF> __device__ __forceinline__ float2 sg_unpack(uint32_t w) {
    if (HALF) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

// N words from an address that is a multiple of 4 N bytes
template <int N> __device__ __forceinline__ void sg_load(const unsigned char* p, uint32_t* w) {
    if constexpr (N == 4) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (N == 2) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = u.x; w[1] = u.y;
    } else {
        w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
}

// FORM: the cache's; QT: query and output type; D: head size; WIDE: 16 query rows instead of 8 (bfloat16 queries, 8-bit forms and
// bfloat16).  Pages hold a multiple of 8 positions.
template <int FORM, typename QT, int D, bool WIDE>
__global__ void __launch_bounds__(32 * SG_MAX_WARPS) attention_single8_kernel(const SingleArgs a) {
    constexpr bool HALF = FORM != C8_BF16;
    constexpr bool TWO = sizeof(QT) == 4 || (!HALF && !WIDE);    // the weights in two numbers
    constexpr bool FLOATQ = sizeof(QT) == 4;                     // the query in two numbers
    constexpr int B = c8_bytes(FORM), ROW = D * B;
    constexpr int KT = ROW <= 64 ? 32 : 16, NK = KT / 4, JT = KT / 8;   // keys of a run, keys of a lane, columns of eight
    constexpr int R = WIDE ? 16 : 8;                             // query rows
    constexpr int NS = D / 16;                                   // products over 16 dimensions
    constexpr int KW = ROW / 16;                                 // words of a key row a lane reads: a quarter
    constexpr int VW = (D / 8 * B + 3) / 4;                      // words of a value row a lane reads: an eighth (D = 80: 2.5 or 5)
    constexpr int NT = D / 8;                                    // dimensions of a value row a lane reads
    extern __shared__ float smem[];

    const int split = blockIdx.x % a.splits, item = blockIdx.x / a.splits;
    const int key_head = blockIdx.y / a.row_blocks, head0 = key_head * a.group + (blockIdx.y % a.row_blocks) * R;
    const int rows = min(R, (key_head + 1) * a.group - head0);
    const int token = a.items ? a.items[item] : item, pos = token >= 0 ? a.positions[token] : -1;
    if (pos < 0) {                                               // (the same for all blocks of a cluster)
        if (a.info) ST_PDL_WAIT();                               // this kernel never ends before the one it was let in by
        return;
    }
    const int* bt = a.kv.table + (size_t)a.slots[a.seq_of_token[token]] * a.kv.max_pages;
    int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    if (a.info) lo = max(lo, a.info[3 * item]);
    const int hi = pos + 1;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    // ---- the query's fragments: dimension of summand k of product s, as the key rows are read
    // pieces of 16 bytes per lane while the row lasts, then 8, then 4
    auto key_byte = [&](int w) -> int {                          // offset of this lane's word w in a key row
        constexpr int full = KW / 4 * 4, two = KW % 4 / 2 * 2;
        if (w < full) return (w / 4) * 64 + t * 16 + (w % 4) * 4;
        if (w < full + two) return full * 16 + t * 8 + (w - full) * 4;
        return (full + two) * 16 + t * 4;
    };
    uint32_t qa[NS][4];
    float fac[WIDE ? 2 : 1];
    {
        const QT* q = (const QT*)a.q + ((size_t)token * a.nh + head0) * D;
#pragma unroll
        for (int half = 0; half < (WIDE ? 2 : 1); ++half) {
            const int r = g + 8 * half;
            const bool ok = r < rows;
            float mul = 1.f;
            float v[NS][4];
            uint32_t amax = 0;
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    // element 4 s + k of the lane's quarter row: a word holds 4 / B of them
                    const int e = 4 * s + k, dim = key_byte(e * B / 4) / B + e % (4 / B);
                    v[s][k] = ok ? to_f32(q[(size_t)r * D + dim]) : 0.f;
                    amax = max(amax, __float_as_uint(v[s][k]) & 0x7fffffffu);
                }
            fac[half] = a.scale_log2;
            if (HALF) {
                amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int ex = min(max((int)(amax >> 23) - 127, -100), 127);
                mul = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
                fac[half] = ldexpf(a.scale_log2, ex - 14);
            }
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const float x = v[s][2 * p] * mul, y = v[s][2 * p + 1] * mul;
                    const uint32_t w = sg_pack<HALF>(x, y);
                    qa[s][2 * p + half] = w;
                    if (!WIDE) {
                        const float2 f = sg_unpack<HALF>(w);
                        qa[s][2 * p + 1] = FLOATQ ? sg_pack<HALF>(x - f.x, y - f.y) : 0u;
                    }
                }
        }
    }
    constexpr int H = WIDE ? 2 : 1;
    float ref[H], sum[H], acc[NT][2 * H];
#pragma unroll
    for (int h = 0; h < H; ++h) { ref[h] = -INFINITY; sum[h] = 0.f; }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int k = 0; k < 2 * H; ++k) acc[i][k] = 0.f;

    const int base0 = lo & ~7, runs = hi > base0 ? (hi - base0 + KT - 1) / KT : 0, stride = W * a.splits;
    // the page and place of this lane's column g (keys) and of its own keys (values, scales) in run i: the first position of
    // an aligned block of eight or four keys, which one page holds
    auto look = [&](int i, int& kpage, int& koff, int& vpage, int& voff) {
        kpage = vpage = -1;
        koff = voff = 0;
        if (i >= runs) return;
        const int b = base0 + i * KT, kk = b + (g >> 1) * NK, vk = b + t * NK;
        if (kk < hi) { kpage = a.kv.page(bt, kk); koff = a.kv.offset(kk, a.kv.page_index(kk)); }
        if (vk < hi) {
            vpage = a.kv.page(bt, vk);
            voff = a.kv.offset(vk, a.kv.page_index(vk));
            if (vpage < 0 && vk + NK > lo && a.kv.status) *a.kv.status = 1;
        }
    };
    uint32_t kw[JT][KW], vw[NK][VW];
    float ks[NK], vs[NK];
    auto load_keys = [&](int page, int off) {
        const uint32_t row = page < 0 ? 0u : a.kv.row0(page, 0, key_head) + off + (g & 1);
        const unsigned char* p = a.kv.pool + (size_t)row * ROW;
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            constexpr int full = KW / 4 * 4, two = KW % 4 / 2 * 2;
            if (page >= 0) {
                const unsigned char* pj = p + 2 * j * ROW;
#pragma unroll
                for (int w = 0; w < full; w += 4) sg_load<4>(pj + key_byte(w), kw[j] + w);
                if constexpr (two > 0) sg_load<2>(pj + key_byte(full), kw[j] + full);
                if constexpr (full + two < KW) sg_load<1>(pj + key_byte(full + two), kw[j] + full + two);
            } else {
#pragma unroll
                for (int w = 0; w < KW; ++w) kw[j][w] = 0u;
            }
        }
    };
    // an eighth of a value row: of every 64 dimensions eight neighbours, then of 32 four, of 16 two
    constexpr int V8 = D / 64, V4 = D % 64 / 32, V2 = D % 32 / 16;
    auto value_dim = [&](int n, int i) -> int {                 // dimension of column n of the i-th product of values
        if (i < 8 * V8) return (i >> 3) * 64 + n * 8 + (i & 7);
        if (i < 8 * V8 + 4 * V4) return 64 * V8 + n * 4 + (i - 8 * V8);
        return 64 * V8 + 32 * V4 + n * 2 + (i - 8 * V8 - 4 * V4);
    };
    auto load_values = [&](int page, int off, int key) {        // key: the first of the lane's keys
        const uint32_t row = page < 0 ? 0u : a.kv.row0(page, 1, key_head) + off;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const unsigned char* p = a.kv.pool + (size_t)(row + k) * ROW;
            if (page >= 0 && key + k >= lo && key + k < hi) {
#pragma unroll
                for (int c = 0; c < V8; ++c) {
                    if constexpr (B == 1) sg_load<2>(p + c * 64 + g * 8, vw[k] + 2 * c);
                    else sg_load<4>(p + c * 128 + g * 16, vw[k] + 4 * c);
                }
                if constexpr (V4) {
                    if constexpr (B == 1) sg_load<1>(p + V8 * 64 + g * 4, vw[k] + 2 * V8);
                    else sg_load<2>(p + V8 * 128 + g * 8, vw[k] + 4 * V8);
                }
                if constexpr (V2) {
                    if constexpr (B == 1) vw[k][VW - 1] = __ldg(reinterpret_cast<const unsigned short*>(p + V8 * 64 + V4 * 32 + g * 2));
                    else sg_load<1>(p + V8 * 128 + V4 * 64 + g * 4, vw[k] + VW - 1);
                }
            } else {
#pragma unroll
                for (int w = 0; w < VW; ++w) vw[k][w] = 0u;
            }
        }
    };
    auto load_scales = [&](int page, int off) {
        if (!HALF || page < 0) {
#pragma unroll
            for (int k = 0; k < NK; ++k) ks[k] = vs[k] = 1.f;
            return;
        }
        const float* k0 = a.kv.scales + a.kv.row0(page, 0, key_head) + off;
        const float* v0 = a.kv.scales + a.kv.row0(page, 1, key_head) + off;
#pragma unroll
        for (int k = 0; k < NK; k += 4) {
            const float4 x = __ldg(reinterpret_cast<const float4*>(k0 + k)), y = __ldg(reinterpret_cast<const float4*>(v0 + k));
            ks[k] = x.x; ks[k + 1] = x.y; ks[k + 2] = x.z; ks[k + 3] = x.w;
            vs[k] = y.x; vs[k + 1] = y.y; vs[k + 2] = y.z; vs[k + 3] = y.w;
        }
    };

    int i = split * W + warp;
    int kpage, koff, vpage, voff, kpage1, koff1, vpage1, voff1;
    look(i, kpage, koff, vpage, voff);
    load_keys(kpage, koff);
    load_values(vpage, voff, base0 + i * KT + t * NK);
    load_scales(vpage, voff);
    look(i + stride, kpage1, koff1, vpage1, voff1);
    for (; i < runs; i += stride) {
        const int key0 = base0 + i * KT + t * NK;                // the lane's keys: key0 .. key0 + NK - 1
        // ---- scores: column n of product j is key (n / 2) NK + 2 j + n % 2 of the run
        float s[JT][4];
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
            for (int x = 0; x < NS; ++x) {
                uint32_t b0, b1;
                if constexpr (HALF) c8_halves<FORM>(kw[j][x], b0, b1);
                else { b0 = kw[j][2 * x]; b1 = kw[j][2 * x + 1]; }
                sg_mma(s[j], qa[x], b0, b1, HALF);
            }
        }
        load_keys(kpage1, koff1);
        // ---- their softmax's numbers: this lane's NK keys of row g (and g + 8)
        float lead = 0.f;                                        // log2 of the largest value scale, rounded up
        if (HALF) {
            float vmax = 0.f;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                if (vpage < 0 || key0 + k < lo || key0 + k >= hi) vs[k] = 0.f;
                vmax = fmaxf(vmax, vs[k]);
            }
            lead = (float)max((int)(__float_as_uint(vmax) >> 23) - 126, -90);
        }
        float corr[H];
        uint32_t pa[KT / 16][4];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            float z[NK], mx = -INFINITY;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                float v = s[k >> 1][2 * h + (k & 1)];
                if (FLOATQ) v += s[k >> 1][2 + (k & 1)];
                if (HALF) v *= ks[k];
                v *= fac[h];
                if (vpage < 0 || key0 + k < lo || key0 + k >= hi) v = -INFINITY;
                z[k] = v;
                mx = fmaxf(mx, v);
            }
            mx += lead;
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            corr[h] = 1.f;
            if (mx > ref[h] + 15.f) {
                const float r = mx - 11.f;
                corr[h] = ar_exp2(ref[h] - r);                   // 0 from "no key yet"
                ref[h] = r;
            }
            const float use = ref[h] == -INFINITY ? 0.f : ref[h];
            float l = 0.f;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                const float p = ar_exp2(z[k] - use);
                l += p;
                z[k] = HALF ? p * vs[k] : p;
            }
            // (a row that is not finite has the scale NaN; where it is masked its weight is zero, not NaN: vs is 0 there)
            sum[h] = sum[h] * corr[h] + l;
#pragma unroll
            for (int m = 0; m < KT / 16; ++m)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const float x = z[4 * m + 2 * p], y = z[4 * m + 2 * p + 1];
                    const uint32_t w = sg_pack<HALF>(x, y);
                    pa[m][2 * p + h] = w;
                    if (!WIDE) {
                        const float2 f = sg_unpack<HALF>(w);
                        pa[m][2 * p + 1] = TWO ? sg_pack<HALF>(x - f.x, y - f.y) : 0u;
                    }
                }
        }
        // ---- weights times values
#pragma unroll
        for (int w = 0; w < VW; ++w) {
            constexpr int PER = 4 / B;                           // dimensions of a word
            uint32_t b[KT / 16][2][4];
#pragma unroll
            for (int m = 0; m < KT / 16; ++m)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const uint32_t x = vw[4 * m + 2 * p][w], y = vw[4 * m + 2 * p + 1][w];
                    if constexpr (HALF) c8_pairs<FORM>(x, y, b[m][p]);
                    else { b[m][p][0] = __byte_perm(x, y, 0x5410); b[m][p][1] = __byte_perm(x, y, 0x7632); }
                }
#pragma unroll
            for (int c = 0; c < PER; ++c) {
                const int n = w * PER + c;
                if (n < NT) {
                    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int m = 0; m < KT / 16; ++m) sg_mma(o, pa[m], b[m][0][c], b[m][1][c], HALF);
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            acc[n][2 * h + k] = acc[n][2 * h + k] * corr[h] + (TWO ? o[k] + o[2 + k] : o[2 * h + k]);
                }
            }
        }
        const int next0 = base0 + (i + stride) * KT + t * NK;
        load_values(vpage1, voff1, next0);
        load_scales(vpage1, voff1);
        vpage = vpage1;
        look(i + 2 * stride, kpage1, koff1, vpage1, voff1);
    }
    // ---- parts to shared memory
    float* s_ref = smem;
    float* s_sum = s_ref + W * R;
    float* s_acc = s_sum + W * R;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        float l = sum[h];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int r = g + 8 * h;
        if (t == 0) { s_ref[warp * R + r] = ref[h]; s_sum[warp * R + r] = l; }
        if (r < rows) {
            float* o = s_acc + ((size_t)warp * R + r) * D;
#pragma unroll
            for (int n = 0; n < NT; ++n) { o[value_dim(2 * t, n)] = acc[n][2 * h]; o[value_dim(2 * t + 1, n)] = acc[n][2 * h + 1]; }
        }
    }
    sg_finish<QT>(a, smem, W, R, rows, D, token, item, head0, key_head);
}

// Blocks, warps and the cluster: n_pairs = items x row blocks of all key heads, each over up to max_keys keys.
struct SingleShape { int splits, warps; };
SingleShape sg_shape(long long n_pairs, int max_keys, int keys_per_run);

template <typename K>
static inline int sg_launch(const char* tag, K kernel, const SingleArgs& a, int warps, size_t smem, int grid_y, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.n_items * a.splits, grid_y);
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (a.splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = a.splits;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (a.info && st_pdl_enabled(tag)) {
        // behind the prefix's kernel, which lets this one's blocks in as its own leave: they work on the tokens' own keys meanwhile
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
    return st_launch_status();
}

template <int FORM, typename QT, int D, bool WIDE>
static int sg_run(SingleArgs a, int max_keys, cudaStream_t s) {
    constexpr int R = WIDE ? 16 : 8, KT = D * c8_bytes(FORM) <= 64 ? 32 : 16;
    a.row_blocks = (a.group + R - 1) / R;
    const int grid_y = a.row_blocks * a.kv.nkv;
    const SingleShape shape = sg_shape((long long)a.n_items * grid_y, max_keys, KT);
    a.splits = shape.splits;
    const size_t smem = (size_t)shape.warps * R * (D + 2) * 4;
    AR_ALLOW_SMEM((attention_single8_kernel<FORM, QT, D, WIDE>), smem);
    return sg_launch("single8", attention_single8_kernel<FORM, QT, D, WIDE>, a, shape.warps, smem, grid_y, s);
}
template <int FORM, typename QT>
static int sg_run(const SingleArgs& a, int max_keys, cudaStream_t s) {
    // 16 rows where a key head has more than eight query heads; a float query needs the other eight for its lower half
    const bool wide = sizeof(QT) == 2 && a.group > 8;
    if constexpr (sizeof(QT) == 2) {
        if (wide) {
            if (a.d == 32) return sg_run<FORM, QT, 32, true>(a, max_keys, s);
            if (a.d == 64) return sg_run<FORM, QT, 64, true>(a, max_keys, s);
            if (a.d == 80) return sg_run<FORM, QT, 80, true>(a, max_keys, s);
            if (a.d == 96) return sg_run<FORM, QT, 96, true>(a, max_keys, s);
            if (a.d == 128) return sg_run<FORM, QT, 128, true>(a, max_keys, s);
            return ST_ERR_BAD_SIZE;
        }
    }
    if (a.d == 32) return sg_run<FORM, QT, 32, false>(a, max_keys, s);
    if (a.d == 64) return sg_run<FORM, QT, 64, false>(a, max_keys, s);
    if (a.d == 80) return sg_run<FORM, QT, 80, false>(a, max_keys, s);
    if (a.d == 96) return sg_run<FORM, QT, 96, false>(a, max_keys, s);
    if (a.d == 128) return sg_run<FORM, QT, 128, false>(a, max_keys, s);
    return ST_ERR_BAD_SIZE;
}

int sg_int8(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s);
int sg_e4m3(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s);
int sg_bf16(const SingleArgs& a, int max_keys, cudaStream_t s);
