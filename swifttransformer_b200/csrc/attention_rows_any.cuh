// Attention over 8-bit caches and shared prefixes in float arithmetic: the kernels that take every head size, page size and type,
// compiled by form in attention_rows_any_{int8,e4m3,wide}.cu.
//
// attention_rows_any_kernel: tiles of query rows (attention_rows.cuh) in float arithmetic.  A block holds a tile's queries, and runs of
// KEYS key and value rows one after the other, in shared memory as floats; scores by 4 x 4 (2 x 2) rows x keys per thread along the
// head's dimensions, the rows' softmax by 256 / ROWS threads each, weights times values by 4 (2) rows x dimensions per thread; both
// products two multiply-adds to an instruction.  Bound by these and by the shared memory's reads (two of 16 bytes per eight
// of them for the scores) where there is much to do, 300 rows of 12 heads (26 us) by the chain from the plan over queries, pages and
// keys to the first product.  ROWS 16 for tiles of at most 16 rows: with 128 only one thread in eight would have work (8 tokens over a
// shared prefix of 1000 keys, 12 heads of 64: 20 us against 27; 32 heads of 128: 56 against 140).
// attention_single_any_kernel: 32 keys to a warp, a lane per key for the scores, lanes along the head's dimensions for the values; for
// single tokens where the kernel of attention_single8.cuh has no instance.  Both visit or use no row that a query does not see: numbers
// that are not finite stay where they are.
#pragma once
#include "attention_single8.cuh"

__device__ __forceinline__ void ar_fma2(float2& d, float2 a, float2 b) {
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 d, {%0, %1};\n\t"
        "fma.rn.f32x2 d, a, b, d;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
        : "+f"(d.x), "+f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}

#define AA_THREADS 256
template <int ROWS> struct AnyShape {
    static constexpr int KEYS = ROWS == 128 ? 32 : 64;
    static constexpr int RPT = ROWS == 128 ? 4 : 2, KPT = ROWS == 128 ? 4 : 2;
    static constexpr int RG = ROWS / RPT, KG = KEYS / KPT;          // groups of rows, of keys (and of dimensions)
    static_assert(RG * KG == AA_THREADS, "");
};
// Blocks that share an SM: what shared memory and the registers of the sums leave room for.  (With two blocks of 128 rows over 8-bit caches
// a prompt of 2000 tokens, 32 heads of 64, takes 815 us instead of 993, but one of 300 tokens of 12 heads, which fills no SM twice, 31
// instead of 26: the registers that two blocks leave are spilled.)
constexpr int aa_blocks(int form, int rows, int dp) { return rows == 16 ? dp <= 64 ? 3 : dp <= 128 ? 2 : 1 : form == C8_F32 && dp <= 64 ? 2 : 1; }
__host__ __device__ inline int aa_stride(int d) { return ((d + 3) & ~3) + 4; }
template <int ROWS> static size_t aa_smem(int d) {
    return (size_t)(ROWS * aa_stride(d) + 2 * AnyShape<ROWS>::KEYS * aa_stride(d) + ROWS * (AnyShape<ROWS>::KEYS + 4)) * 4;
}

// four neighbouring elements of a cache row as they lie in memory, and as floats
template <int FORM> struct AnyRaw {
    using type = uint32_t;
    static __device__ __forceinline__ float4 floats(uint32_t w) {
        uint32_t h[2];
        c8_halves<FORM == C8_E4M3 ? C8_E4M3 : C8_INT8>(w, h[0], h[1]);
        const float2 x = sg_unpack<true>(h[0]), y = sg_unpack<true>(h[1]);
        return make_float4(x.x, x.y, y.x, y.y);
    }
};
template <> struct AnyRaw<C8_F32> {
    using type = float4;
    static __device__ __forceinline__ float4 floats(float4 v) { return v; }
};

template <int FORM, typename QT, int ROWS, int DP>
__global__ void __launch_bounds__(AA_THREADS, aa_blocks(FORM, ROWS, DP)) attention_rows_any_kernel(const RowArgs a) {
    using S = AnyShape<ROWS>;
    constexpr int KEYS = S::KEYS, RPT = S::RPT, KPT = S::KPT, RG = S::RG, KG = S::KG;
    constexpr int DT = (DP + 4 * KG - 1) / (4 * KG);               // pieces of four dimensions per thread
    constexpr int TPR = AA_THREADS / ROWS;                         // threads of a row's softmax
    extern __shared__ __align__(16) float aa_smem_raw[];
    __shared__ uint32_t s_row[KEYS];
    __shared__ float s_ks[KEYS], s_vs[KEYS];
    __shared__ int s_pos[ROWS], s_token[ROWS], s_odd;
    __shared__ float s_corr[ROWS];
    const int d = a.d, ld = aa_stride(d), nv = (d + 3) / 4;
    float* sq = aa_smem_raw;
    float* sk = sq + ROWS * ld;
    float* sv = sk + KEYS * ld;
    float* sp = sv + KEYS * ld;
    constexpr int LP = KEYS + 4;
    const int tid = threadIdx.x, rg = tid / KG, kg = tid % KG, g = a.plan.group;
    const uint32_t to_values = (uint32_t)a.kv.nkv * a.kv.page_size;
    // four elements of a query row at once
    const bool wide = d % 4 == 0 && a.q_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;
    ST_PDL_TRIGGER();
    RowWalk walk;
    walk.begin(a.plan, blockIdx.x);
    RowPiece pc;
    while (walk.next(a.plan, pc)) {
        const int rows = pc.t.n_tok * g;
        __syncthreads();                                            // the piece before is done with shared memory
        for (int r = tid; r < ROWS; r += AA_THREADS) {
            const int token = r < rows ? (a.plan.items ? a.plan.items[pc.t.first + r / g] : pc.t.first + r / g) : -1;
            s_token[r] = token;
            s_pos[r] = token >= 0 ? a.positions[token] : -1;
        }
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < ROWS * nv; i += AA_THREADS) {
            const int r = i / nv, e = (i - r * nv) * 4;
            const int token = s_token[r];
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (token >= 0) {
                const QT* q = (const QT*)a.q + (size_t)token * a.q_stride + (size_t)(pc.head * g + r % g) * d + e;
                if (wide) {
                    x = load4(q);
                } else {
                    x.x = to_f32(q[0]);
                    if (e + 1 < d) x.y = to_f32(q[1]);
                    if (e + 2 < d) x.z = to_f32(q[2]);
                    if (e + 3 < d) x.w = to_f32(q[3]);
                }
                x.x *= a.scale_log2; x.y *= a.scale_log2; x.z *= a.scale_log2; x.w *= a.scale_log2;
            }
            store4(sq + r * ld + e, x);
        }
        const RowTable table = pc.t.seq < 0 ? ar_table<true>(a, pc.t) : ar_table<false>(a, pc.t);
        float ref = -INFINITY, sum = 0.f;                           // of row tid / TPR
        float2 acc[RPT][DT][2];
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int c = 0; c < DT; ++c) acc[i][c][0] = acc[i][c][1] = make_float2(0.f, 0.f);
        const int k_begin = (pc.t.key_lo & ~(AR_CHUNK - 1)) + pc.chunk0 * AR_CHUNK;
        const int k_end = min(k_begin + pc.chunks * AR_CHUNK, pc.t.key_hi);
        // key k0 + tid (tid < KEYS): its page, looked up while the run before is worked on, then its row and scales
        int page = -1;
        bool wanted = false;
        auto ask = [&](int k0) {
            if (tid >= KEYS) return;                                // (whole warps)
            const int key = k0 + tid, index = a.kv.page_index(key);
            const int* const from = ar_row_of<true>(a, pc.t, table, key, key >= pc.t.key_lo && key < k_end);
            wanted = from != nullptr;
            page = wanted && index < a.kv.max_pages ? __ldg(from + index) : -1;
        };
        uint32_t row_of = 0xffffffffu;
        float ks_of = 1.f, vs_of = 1.f;
        auto resolve = [&](int k0) {
            const int key = k0 + tid;
            row_of = 0xffffffffu;
            ks_of = vs_of = 1.f;
            if (!wanted) return;
            if ((unsigned)page >= (unsigned)a.kv.num_pages) {
                if (pc.t.seq < 0 || ar_needed(a, pc.t, key)) *a.kv.status = 1;
                return;
            }
            row_of = a.kv.row0(page, 0, pc.head) + a.kv.offset(key, a.kv.page_index(key));
            if (FORM < C8_BF16) { ks_of = __ldg(a.kv.scales + row_of); vs_of = __ldg(a.kv.scales + row_of + to_values); }
        };
        ask(k_begin);
        resolve(k_begin);
        for (int k0 = k_begin; k0 < k_end; k0 += KEYS) {
            __syncthreads();
            if (tid == 0) s_odd = 0;
            if (tid < KEYS) { s_row[tid] = row_of; s_ks[tid] = ks_of; s_vs[tid] = vs_of; }
            __syncthreads();
            ask(k0 + KEYS);
            // rows as floats; what lies past d or has no key is zero.  Two pieces' loads are under way together.
            bool odd = false;
            if (FORM != C8_BF16 && d % 4 == 0) {
                using Raw = typename AnyRaw<FORM>::type;
                const Raw* keys = reinterpret_cast<const Raw*>(a.kv.pool);
                for (int i0 = tid; i0 < KEYS * nv; i0 += 2 * AA_THREADS) {
                    Raw k[2], v[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int i = i0 + c * AA_THREADS, j = i / nv;
                        const uint32_t row = i < KEYS * nv ? s_row[j] : 0xffffffffu;
                        k[c] = v[c] = Raw{};
                        if (row != 0xffffffffu) {
                            k[c] = __ldg(keys + (size_t)row * nv + (i - j * nv));
                            v[c] = __ldg(keys + (size_t)(row + to_values) * nv + (i - j * nv));
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int i = i0 + c * AA_THREADS, j = i / nv;
                        if (i >= KEYS * nv) continue;
                        const float4 x = AnyRaw<FORM>::floats(k[c]);
                        float4 y = AnyRaw<FORM>::floats(v[c]);
                        if (FORM < C8_BF16) {
                            const float s = s_vs[j];
                            y.x *= s; y.y *= s; y.z *= s; y.w *= s;
                        }
                        odd |= !(isfinite(y.x) && isfinite(y.y) && isfinite(y.z) && isfinite(y.w));
                        store4(sk + j * ld + (i - j * nv) * 4, x);
                        store4(sv + j * ld + (i - j * nv) * 4, y);
                    }
                }
            } else {
                for (int i = tid; i < KEYS * nv * 4; i += AA_THREADS) {
                    const int j = i / (nv * 4), e = i - j * nv * 4;
                    const uint32_t row = e < d ? s_row[j] : 0xffffffffu;
                    float k = 0.f, v = 0.f;
                    if (row != 0xffffffffu) {
                        k = c8_value<FORM>(a.kv.pool, (size_t)row * d + e);
                        v = c8_value<FORM>(a.kv.pool, (size_t)(row + to_values) * d + e) * s_vs[j];
                    }
                    odd |= !isfinite(v);
                    sk[j * ld + e] = k;
                    sv[j * ld + e] = v;
                }
            }
            if (odd) s_odd = 1;
            resolve(k0 + KEYS);
            __syncthreads();
            // ---- scores
            if (rg < rows) {
                float2 z[RPT][KPT];
#pragma unroll
                for (int i = 0; i < RPT; ++i)
#pragma unroll
                    for (int j = 0; j < KPT; ++j) z[i][j] = make_float2(0.f, 0.f);
                for (int e = 0; e < nv * 4; e += 4) {
                    float4 x[RPT], y[KPT];
#pragma unroll
                    for (int i = 0; i < RPT; ++i) x[i] = load4(sq + (rg + RG * i) * ld + e);
#pragma unroll
                    for (int j = 0; j < KPT; ++j) y[j] = load4(sk + (kg + KG * j) * ld + e);
#pragma unroll
                    for (int i = 0; i < RPT; ++i)
#pragma unroll
                        for (int j = 0; j < KPT; ++j) {
                            ar_fma2(z[i][j], make_float2(x[i].x, x[i].y), make_float2(y[j].x, y[j].y));
                            ar_fma2(z[i][j], make_float2(x[i].z, x[i].w), make_float2(y[j].z, y[j].w));
                        }
                }
#pragma unroll
                for (int i = 0; i < RPT; ++i) {
                    const int r = rg + RG * i, pos = s_pos[r];
                    const int low = a.window > 0 ? pos - a.window + 1 : 0;
#pragma unroll
                    for (int j = 0; j < KPT; ++j) {
                        const int jj = kg + KG * j, key = k0 + jj;
                        const bool seen = s_row[jj] != 0xffffffffu && key <= pos && key >= low;
                        sp[r * LP + jj] = seen ? (z[i][j].x + z[i][j].y) * s_ks[jj] : -INFINITY;
                    }
                }
            }
            __syncthreads();
            // ---- softmax of row tid / TPR
            {
                const int r = tid / TPR, sub = tid % TPR;
                constexpr int N = KEYS / TPR;
                float z[N], mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    z[j] = r < rows ? sp[r * LP + sub + TPR * j] : -INFINITY;
                    mx = fmaxf(mx, z[j]);
                }
#pragma unroll
                for (int o = TPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const float m = fmaxf(ref, mx), use = m == -INFINITY ? 0.f : m;
                const float corr = ref == -INFINITY ? 0.f : exp2f(ref - m);
                float l = 0.f;
                const bool odd = s_odd != 0;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float p = exp2f(z[j] - use);
                    l += p;
                    // a weight of zero stands for a key that is hidden, where a value is not finite: one that is seen weighs a little
                    sp[r * LP + sub + TPR * j] = odd && p == 0.f && z[j] != -INFINITY ? 1e-45f : p;
                }
                sum = sum * corr + l;
                ref = m;
                if (sub == 0) s_corr[r] = corr;
            }
            __syncthreads();
            // ---- weights times values: rows rg + RG i, dimensions 4 (kg + KG c) .. + 3
            if (rg < rows) {
                const bool guard = s_odd != 0;                      // a hidden key's weight must not meet a value that is not finite
#pragma unroll
                for (int i = 0; i < RPT; ++i) {
                    const float corr = s_corr[rg + RG * i];
#pragma unroll
                    for (int c = 0; c < DT; ++c)
#pragma unroll
                        for (int h = 0; h < 2; ++h) { acc[i][c][h].x *= corr; acc[i][c][h].y *= corr; }
                }
                const int n_keys = min(KEYS, k_end - k0);
#pragma unroll 4
                for (int j = 0; j < n_keys; ++j) {
                    float p[RPT];
#pragma unroll
                    for (int i = 0; i < RPT; ++i) p[i] = sp[(rg + RG * i) * LP + j];
#pragma unroll
                    for (int c = 0; c < DT; ++c) {
                        const int e = 4 * (kg + KG * c);
                        if (e >= nv * 4) continue;
                        const float4 v = load4(sv + j * ld + e);
#pragma unroll
                        for (int i = 0; i < RPT; ++i) {
                            if (guard && p[i] == 0.f) continue;
                            ar_fma2(acc[i][c][0], make_float2(p[i], p[i]), make_float2(v.x, v.y));
                            ar_fma2(acc[i][c][1], make_float2(p[i], p[i]), make_float2(v.z, v.w));
                        }
                    }
                }
            }
        }
        // ---- the piece's sums: out, or into its slot
        {
            const int sub = tid % TPR;
#pragma unroll
            for (int o = TPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            __syncthreads();
            float* s_sum = sp;
            if (sub == 0) { s_sum[tid / TPR] = sum; s_sum[ROWS + tid / TPR] = ref; }
            __syncthreads();
            const bool direct = a.direct && pc.whole;
            const size_t slot = (size_t)ar_slot(a, pc, blockIdx.x) * AR_ROWS;
            if (!direct)
                for (int r = tid; r < rows; r += AA_THREADS) { a.parts.r[slot + r] = s_sum[ROWS + r]; a.parts.l[slot + r] = s_sum[r]; }
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
                const int r = rg + RG * i;
                if (r >= rows) continue;
                const float l = s_sum[r], inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                for (int c = 0; c < DT; ++c) {
                    const int e = 4 * (kg + KG * c);
                    const float o[4] = {acc[i][c][0].x, acc[i][c][0].y, acc[i][c][1].x, acc[i][c][1].y};
                    if (d % 4 == 0 && !direct) {
                        if (e < d) store4(a.parts.o + (slot + r) * d + e, make_float4(o[0], o[1], o[2], o[3]));
                        continue;
                    }
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        if (e + h >= d) continue;
                        if (!direct) a.parts.o[(slot + r) * d + e + h] = o[h];
                        else if (s_pos[r] >= 0)
                            ((QT*)a.out)[((size_t)s_token[r] * a.plan.nh + pc.head * g + r % g) * d + e + h] = from_f32<QT>(o[h] * inv);
                    }
                }
            }
        }
    }
}

// ---- single tokens, anything ----------------------------------------------------------------------------------------
template <int FORM, typename QT>
__global__ void __launch_bounds__(128) attention_single_any_kernel(const SingleArgs a) {
    extern __shared__ __align__(128) float smem[];
    const int split = blockIdx.x % a.splits, item = blockIdx.x / a.splits, head = blockIdx.y, key_head = head / a.group, d = a.d;
    const int token = a.items ? a.items[item] : item, pos = token >= 0 ? __ldg(a.positions + token) : -1;
    const int seq = token >= 0 ? __ldg(a.seq_of_token + token) : 0;
    if (pos < 0) {
        if (a.info) ST_PDL_WAIT();
        return;
    }
    const int* bt = a.kv.table + (size_t)__ldg(a.slots + seq) * a.kv.max_pages;
    const SingleSpan span = sg_span(a, item, pos);
    const int lo = span.lo, last = span.hi - 1;
    if (last < pos && a.kv.status) *a.kv.status = 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
    const uint32_t to_values = (uint32_t)a.kv.nkv * a.kv.page_size;
    float* sq = smem;                                              // the query row, scaled, then zeros up to a multiple of four
    float* parts = smem + ((d + 3) & ~3);
    for (int e = threadIdx.x; e < ((d + 3) & ~3); e += blockDim.x)
        sq[e] = e < d ? to_f32(((const QT*)a.q)[((size_t)token * a.nh + head) * d + e]) * a.scale_log2 : 0.f;
    __syncthreads();
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    float ref = -INFINITY, sum = 0.f;
    for (int b = lo + (split * W + warp) * 32; b <= last; b += a.splits * W * 32) {
        uint32_t row = 0xffffffffu;
        float ks = 1.f, vs = 1.f;
        if (b + lane <= last) {
            const int page = a.kv.page(bt, b + lane);
            if (page >= 0) {
                row = a.kv.row0(page, 0, key_head) + a.kv.offset(b + lane, a.kv.page_index(b + lane));
                if (FORM < C8_BF16) { ks = __ldg(a.kv.scales + row); vs = __ldg(a.kv.scales + row + to_values); }
            } else if (a.kv.status) {
                *a.kv.status = 1;
            }
        }
        // a lane has a key of its own for the scores, dimensions lane, lane + 32, ... for the values
        float z = -INFINITY;
        const int n = min(32, last - b + 1);
        if (row != 0xffffffffu) {
            float dot = 0.f;
            if (FORM != C8_BF16 && d % 4 == 0) {
                using Raw = typename AnyRaw<FORM>::type;
                const Raw* key = reinterpret_cast<const Raw*>(a.kv.pool) + (size_t)row * (d / 4);
#pragma unroll 8
                for (int e = 0; e < d / 4; ++e) {
                    const float4 x = AnyRaw<FORM>::floats(__ldg(key + e)), y = load4(sq + 4 * e);
                    dot += (x.x * y.x + x.y * y.y) + (x.z * y.z + x.w * y.w);
                }
            } else {
#pragma unroll 4
                for (int e = 0; e < d; ++e) dot += sq[e] * c8_value<FORM>(a.kv.pool, (size_t)row * d + e);
            }
            z = dot * ks;
        }
        const float mx = warp_max(z), m = fmaxf(ref, mx), use = m == -INFINITY ? 0.f : m;
        const float corr = ref == -INFINITY ? 0.f : exp2f(ref - m), p = exp2f(z - use);
        ref = m;
        sum = sum * corr + p;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= corr;
        const float w = p * vs;
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
            const uint32_t r = __shfl_sync(0xffffffffu, row, j);
            const float wj = __shfl_sync(0xffffffffu, w, j);
            if (r != 0xffffffffu) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (lane + 32 * i < d) acc[i] += wj * c8_value<FORM>(a.kv.pool, (size_t)(r + to_values) * d + lane + 32 * i);
            }
        }
    }
    sum = warp_sum(sum);
    if (lane == 0) { parts[warp] = ref; parts[W + warp] = sum; }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < d) parts[2 * W + warp * d + lane + 32 * i] = acc[i];
    sg_finish<QT>(a, parts, W, 1, 1, d, token, pos, item, head, key_head);
}

template <int FORM, typename QT> static int aa_single(SingleArgs a, int max_keys, cudaStream_t s) {
    const SingleShape shape = sg_shape((long long)a.n_items * a.nh, max_keys, 32);
    a.splits = shape.splits;
    a.row_blocks = 1;
    const int warps = shape.warps < 4 ? shape.warps : 4;
    return sg_launch("single_any", attention_single_any_kernel<FORM, QT>, a, dim3((unsigned)a.n_items * a.splits, a.nh), warps,
                     ((size_t)warps * (a.d + 2) + ((a.d + 3) & ~3)) * 4, s);
}

template <int FORM, typename QT, int ROWS> static int aa_rows(const RowArgs& a, cudaStream_t s) {
    const size_t smem = aa_smem<ROWS>(a.d);
    const int grid = a.plan.ctas;
    if (a.d <= 64) {
        AR_ALLOW_SMEM((attention_rows_any_kernel<FORM, QT, ROWS, 64>), aa_smem<ROWS>(64));
        attention_rows_any_kernel<FORM, QT, ROWS, 64><<<grid, AA_THREADS, smem, s>>>(a);
    } else if (a.d <= 128) {
        AR_ALLOW_SMEM((attention_rows_any_kernel<FORM, QT, ROWS, 128>), aa_smem<ROWS>(128));
        attention_rows_any_kernel<FORM, QT, ROWS, 128><<<grid, AA_THREADS, smem, s>>>(a);
    } else {
        AR_ALLOW_SMEM((attention_rows_any_kernel<FORM, QT, ROWS, 256>), aa_smem<ROWS>(256));
        attention_rows_any_kernel<FORM, QT, ROWS, 256><<<grid, AA_THREADS, smem, s>>>(a);
    }
    return st_launch_status();
}
template <int FORM, typename QT> static int aa_rows(const RowArgs& a, int max_rows, cudaStream_t s) {
    return max_rows <= 16 ? aa_rows<FORM, QT, 16>(a, s) : aa_rows<FORM, QT, 128>(a, s);
}
