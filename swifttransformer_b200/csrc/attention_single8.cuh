// Attention of single query tokens over paged caches in 8 and 16 bits, of all keys or of those behind a shared prefix.  A unit is a
// (token, key head, up to eight of its query heads).  Few keys: a block or a cluster of blocks per unit, whose warps take its runs of
// keys in turn and join their parts through shared memory.  Many keys: all units' runs are one line that is cut evenly (SingleLine).
//
// Mathematics: s_j = (q . c_j) ks_j, o = sum_j p_j vs_j c'_j / sum_j p_j with the codes c, c' and the rows' scales ks, vs: the
// scales leave both products, whose operands are then exact in 16 bits: codes of either 8-bit form are halves; a bfloat16 query
// is scaled by a power of two per row, so that its largest element lies in [2^14, 2^15), and is a half unless an element is
// 2^-29 of that or less; a float query is the sum of two halves (22 bits; the rest, 2^-23 of an element, is below what 32-bit
// sums round away).  The weights are p_j vs_j in a half of 2^-11, for float queries and for up to four heads over bfloat16 caches in
// two numbers.  Sums are float.
//
// Products are mma.sync (m16n8k16) with sixteen keys, then sixteen dimensions, on the row side, whose operand takes four
// registers, all of them data, and the query heads as the eight columns: S^T = K Q^T, O^T += V^T P^T.  (With the heads on the row side
// half of that operand is zeros, which have to be moved into place: 630 instructions for 16 keys of 128 dimensions; this
// way 300.)  Two numbers of a head are columns h and h + 4.
//
// p_j = 2^(s_j - R): R follows the largest of s_j + log2 vs_j in steps: it moves when that exceeds R + 15, and then to 11 below, so
// that p_j vs_j stays below 2^15 and what is 2^-24 of the largest still has a half's full precision.  For float queries the values' sums
// of a run are formed in fresh accumulators and added to the running ones with a float add each: tensor cores cut
// what they add to a large sum.
//
// Layout.  A warp walks runs of KT = 32 keys (16 where rows are longer than 128 bytes), each four aligned blocks of KT / 4 keys within a
// page, which come by 16-byte asynchronous copies into a ring of its own in shared memory, one or two runs ahead: 8 KB a warp
// under way, 100 to 140 KB an SM.  Lane (g, t) = (lane / 4, lane % 4) takes of the key rows that are rows g and g + 8 of a product a
// quarter in pieces of 16 bytes (the order of the summed dimensions is free, the query's is the same), and of the values of KT/4
// neighbouring keys an eighth of the row.  Keys are dealt to rows so that lane t's values are block t's and each lane looks up
// one page per run; the weights change lanes in one transposition (movmatrix) per 8 x 8.  Rows are kept permuted (sg_key_at,
// sg_value_at) so that lanes that read together hit different banks.
//
// Many keys: bound by memory and the issue of instructions together: 4.5 TB/s at 57 % of the issue slots (64 requests of 500 to 1500
// keys, 32 heads of 64, e4m3: 60 us), 3.4 TB/s where 4 of the 8 columns are used (4 requests of 30000 keys, 4 heads of 128: 35 us),
// 2.4 TB/s for float queries, whose products are twice as many (27 us).  Few: by the chain of loads to the first keys and the join
// (one request of 1000 keys: 7 us).
#pragma once
#include "attention_rows.cuh"

#define SG_MAX_WARPS 16
#define SG_LINE_ITEMS 1024           // tokens of a call that is dealt out as one line
#define SG_LINE_WARPS 4              // warps of its blocks
// by the bytes of a row: keys of a run, runs of a warp's ring, and blocks of four warps on an SM, as their registers and rings allow
__host__ __device__ constexpr int sg_run_keys(int row) { return row <= 128 ? 32 : 16; }
__host__ __device__ constexpr int sg_stages(int row) { return row <= 80 ? 3 : 2; }
__host__ __device__ constexpr int sg_line_blocks(int row) { return row <= 64 ? 4 : 3; }
#define SG_SMEM (200 * 1024)         // the most shared memory of a block that has one unit; its parts take less than its rings may
#define SG_JOIN 512                  // the most threads that join a row's parts

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
    // calls dealt out as one line: its walkers' parts (as in RowParts, R rows to a slot), and the first and last walker of every
    // (key head and row block, token)
    RowParts line;
    int* span;
    int walkers;                 // 0: no line
};

// The keys [lo, hi) that a token reads itself: those of its window behind the `shared` ones, as far as the table reaches (what lies past it
// has no page).  lo <= hi <= reach also where there are none, as for a window that lies wholly past the table: warps form the
// keys of their first runs before they know that there are none, and these stay in an int (c8_reach).
struct SingleSpan { int lo, hi; };
__host__ __device__ inline SingleSpan sg_span(int pos, int window, int shared, int reach) {
    const int hi = (pos < reach - 1 ? pos : reach - 1) + 1, first = window > 0 && pos >= window ? pos - window + 1 : 0;
    const int lo = first > shared ? first : shared;
    return SingleSpan{lo < hi ? lo : hi, hi};
}

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

// The parts of a token's shared keys: rows row, row + AR_ROWS, ... (n of them) of a.parts, for the key head's first query head.
struct SharedParts { size_t row; int n; };
__device__ __forceinline__ SharedParts sg_shared_parts(const SingleArgs& a, int item, int key_head, int pos) {
    if (!a.info) return SharedParts{0, 0};
    const int tile = a.info[3 * item + 1], place = a.info[3 * item + 2];
    const RowTile t = ar_tile(a.plan, tile);
    if (a.window > 0 && pos >= 0 && max(0, pos - a.window + 1) < t.key_lo && threadIdx.x == 0) *a.kv.status = 1;   // keys that the plan left out
    const int n = ar_chunks(t);
    if (n == 0) return SharedParts{0, 0};
    int c0, c1;
    ar_walkers(a.plan, t, key_head, n, c0, c1);
    return SharedParts{(size_t)(tile * a.plan.nkv + key_head + c0) * AR_ROWS + place * a.group, c1 - c0 + 1};
}

// The warps' parts of R rows x D, then the cluster's, then the prefix's, to the output.  smem: W x R x (D + 2) floats: (R, l) of each
// warp and row, then O.  `rows` of the R are real; head0 is the first one's query head.
template <typename QT>
__device__ __forceinline__ void sg_finish(const SingleArgs& a, float* smem, int W, int R, int rows, int D, int token, int pos, int item,
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
    SharedParts shared = sg_shared_parts(a, item, key_head, pos);
    if (a.info) ST_PDL_WAIT();                         // the prefix's parts are complete
    QT* out = (QT*)a.out + ((size_t)token * a.nh + head0) * D;
    for (int i = threadIdx.x + rank * blockDim.x; i < rows * D; i += blockDim.x * a.splits) {
        const int r = i / D;
        const size_t row = shared.row + (head0 - key_head * a.group) + r;
        float m = -INFINITY, l = 0.f, o = 0.f;
        for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.splits > 1 ? sg_remote(ref + r, s) : ref[r]);
#pragma unroll 8
        for (int p = 0; p < shared.n; ++p) m = fmaxf(m, __ldcg(a.parts.r + row + (size_t)p * AR_ROWS));
        for (int s = 0; s < a.splits; ++s) {
            const float w = ar_weight(a.splits > 1 ? sg_remote(ref + r, s) : ref[r], m);
            l += w * (a.splits > 1 ? sg_remote(sum + r, s) : sum[r]);
            o += w * (a.splits > 1 ? sg_remote(acc + i, s) : acc[i]);
        }
#pragma unroll 8
        for (int p = 0; p < shared.n; ++p) {
            const size_t at = row + (size_t)p * AR_ROWS;
            const float w = ar_weight(__ldcg(a.parts.r + at), m);
            l += w * __ldcg(a.parts.l + at);
            o += w * __ldcg(a.parts.o + at * D + (i - r * D));
        }
        out[i] = from_f32<QT>(l == 0.f ? 0.f : o / l);   // no key at all: zeros
    }
    if (a.splits > 1) sg_cluster_sync();               // nobody leaves while others read here
}

// c = a b (+ c)
template <bool HALF, bool ADD> __device__ __forceinline__ void sg_mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    const float z0 = ADD ? c[0] : 0.f, z1 = ADD ? c[1] : 0.f, z2 = ADD ? c[2] : 0.f, z3 = ADD ? c[3] : 0.f;
    if (HALF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
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

// N words of shared memory from an address that is a multiple of 4 N bytes
template <int N> __device__ __forceinline__ void sg_load(uint32_t p, uint32_t* w) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(p));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "r"(p));
    else
        asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(w[0]) : "r"(p));
}
__device__ __forceinline__ uint32_t sg_load2(uint32_t p) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(v) : "r"(p));
    return v;
}
__device__ __forceinline__ void sg_copy16(uint32_t dst, const void* src, bool ok) {      // zeros where not ok
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
// Where byte b (the first of 16) of row k of block t is kept, in blocks of N rows.  Keys: eight lanes read 64 bytes each of two
// neighbouring rows; with rows of 128 bytes or more every second row has its halves of 128 bytes exchanged.  Values: lanes
// of all four blocks read the same bytes of row k of theirs; the blocks' rows lie a multiple of 128 bytes apart, so block t's
// pieces are moved by t.
template <int ROW> __device__ __forceinline__ uint32_t sg_key_at(int row, int b) {
    return row * ROW + (ROW % 128 == 0 ? b ^ ((row & 1) << 6) : b);
}
template <int ROW, int N> __device__ __forceinline__ uint32_t sg_value_at(int t, int k, int b) {
    if (ROW == 64) return (t * N + (k ^ (t & 1))) * ROW + (b ^ ((t >> 1) << 5));
    return (t * N + k) * ROW + (ROW % 128 == 0 ? b ^ (t << 5) : b);
}

// Calls of many keys are dealt out as one line: the runs of all tokens one behind the other, once per key head and row block, cut into
// equal parts, one per warp, however unequal the tokens are (blocks that each had one token's keys left the device a third
// empty at 64 requests of 500 to 1500 tokens).  Every block adds up the tokens' runs itself.
template <bool LINE> struct SingleLine {
    int length, total, run;
    int before[LINE ? SG_LINE_ITEMS + 1 : 1];
};
__device__ __forceinline__ SingleSpan sg_span(const SingleArgs& a, int item, int pos) {
    return sg_span(pos, a.window, a.info ? a.info[3 * item] : 0, a.kv.reach);
}
template <int KT> __device__ __forceinline__ int sg_runs(const SingleArgs& a, int item, int pos) {     // of a token's own keys
    const SingleSpan k = sg_span(a, item, pos);
    return k.hi > k.lo ? (k.hi - (k.lo & ~7) + KT - 1) / KT : 0;
}
template <int KT> __device__ __forceinline__ void sg_line_begin(const SingleArgs& a, SingleLine<true>& s) {
    for (int i = threadIdx.x; i < a.n_items; i += blockDim.x) {
        const int token = a.items ? a.items[i] : i, pos = token >= 0 ? a.positions[token] : -1;
        s.before[i + 1] = sg_runs<KT>(a, i, pos);
        if (pos >= a.kv.reach && a.kv.status) *a.kv.status = 1;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        int sum = 0;
        for (int i = 0; i < a.n_items; i += 32) {
            int v = i + threadIdx.x < a.n_items ? s.before[i + threadIdx.x + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (threadIdx.x >= o) v += u;
            }
            v += sum;
            if (i + threadIdx.x < a.n_items) s.before[i + threadIdx.x + 1] = v;
            sum = __shfl_sync(0xffffffffu, v, 31);
        }
        if (threadIdx.x == 0) {
            s.before[0] = 0;
            s.length = sum;
            s.total = sum * a.row_blocks * a.kv.nkv;
            s.run = max(1, (s.total + a.walkers - 1) / a.walkers);
        }
    }
    __syncthreads();
}
// the item whose runs hold run r of the line
__device__ __forceinline__ int sg_line_find(const SingleLine<true>& s, int n_items, int r) {
    int lo = 0, hi = n_items - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s.before[mid] <= r) lo = mid; else hi = mid - 1;
    }
    return lo;
}
// A block per (unit, row): the parts that several walkers left, and those of shared keys, four dimensions a thread, the parts dealt out
// to the threads that remain.
template <typename QT, int KT>
__global__ void __launch_bounds__(SG_JOIN) attention_single8_join_kernel(const SingleArgs a, int R) {
    __shared__ float s_max[SG_JOIN / 32], s_l[SG_JOIN];
    __shared__ float4 s_o[SG_JOIN];
    const int unit = blockIdx.x, part = unit / a.n_items, item = unit - part * a.n_items, d = a.d, r = blockIdx.y;
    const int key_head = part / a.row_blocks, head = key_head * a.group + (part % a.row_blocks) * R + r;
    if (head >= (key_head + 1) * a.group) return;                // (row 0 of the unit is there and waits)
    const int token = a.items ? a.items[item] : item, pos = token >= 0 ? a.positions[token] : -1;
    const SharedParts shared = sg_shared_parts(a, item, key_head, pos);
    const size_t shared_row = shared.row + (head - key_head * a.group);
    const bool own = pos >= 0 && sg_runs<KT>(a, item, pos) > 0;
    ST_PDL_WAIT();                                               // by all, so that what follows this kernel follows the one before it too
    if (pos < 0) return;
    const int c0 = own ? __ldcg(a.span + 2 * unit) : 0, c1 = own ? __ldcg(a.span + 2 * unit + 1) : -1;
    if (!a.info && own && c0 == c1) return;                             // one walker had it all and has stored it
    const int lanes = d / 4, groups = blockDim.x / lanes, mine = threadIdx.x / lanes, e = threadIdx.x % lanes * 4;
    const int n_own = c1 - c0 + 1, n = n_own + shared.n;
    float m = -INFINITY;
    for (int p = threadIdx.x; p < n; p += blockDim.x)
        m = fmaxf(m, p < n_own ? __ldcg(a.line.r + (size_t)(unit + c0 + p) * R + r) : __ldcg(a.parts.r + shared_row + (size_t)(p - n_own) * AR_ROWS));
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int i = 0; i < blockDim.x / 32; ++i) m = fmaxf(m, s_max[i]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine < groups) {
#pragma unroll 8
        for (int p = mine; p < n; p += groups) {
            const RowParts& from = p < n_own ? a.line : a.parts;
            const size_t at = p < n_own ? (size_t)(unit + c0 + p) * R + r : shared_row + (size_t)(p - n_own) * AR_ROWS;
            const float w = ar_weight(__ldcg(from.r + at), m);
            const float4 v = load4_cg(from.o + at * d + e);
            l += w * __ldcg(from.l + at);
            o.x += w * v.x; o.y += w * v.y; o.z += w * v.z; o.w += w * v.w;
        }
    }
    s_l[threadIdx.x] = l;
    s_o[threadIdx.x] = o;
    __syncthreads();
    if (mine == 0) {
        for (int k = 1; k < groups; ++k) {
            l += s_l[k * lanes + threadIdx.x];
            o = add4(o, s_o[k * lanes + threadIdx.x]);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        store4((QT*)a.out + ((size_t)token * a.nh + head) * d + e, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
}

__device__ __forceinline__ uint32_t sg_transpose(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
    return d;
}

// FORM: the cache's; QT: query and output type; D: head size; TWO: weights (and float queries) in two numbers, four heads to a block
// instead of eight.  Pages hold a multiple of 8 positions.
// LINE: see SingleLine.
template <int FORM, typename QT, int D, bool TWO, bool LINE>
__global__ void __launch_bounds__(LINE ? 32 * SG_LINE_WARPS : 32 * SG_MAX_WARPS, LINE ? sg_line_blocks(D * c8_bytes(FORM)) : 1) attention_single8_kernel(const SingleArgs a) {
    constexpr bool HALF = FORM != C8_BF16;
    constexpr bool FLOATQ = sizeof(QT) == 4;
    static_assert(TWO || !FLOATQ, "");
    constexpr int B = c8_bytes(FORM), ROW = D * B;
    constexpr int KT = sg_run_keys(ROW), NK = KT / 4, MT = KT / 16;      // keys of a run, keys of a lane, products over 16 keys
    constexpr int STAGES = sg_stages(ROW);
    constexpr int R = TWO ? 4 : 8;                               // query heads
    constexpr int NS = D / 16;                                   // products over 16 dimensions
    constexpr int KW = ROW / 16;                                 // words of a key row a lane reads: a quarter
    constexpr int VW = (D / 8 * B + 3) / 4;                      // words of a value row a lane reads: an eighth (D = 80: 2.5 or 5)
    constexpr int NT = D / 8;                                    // dimensions of a value row a lane reads
    constexpr int BLOCK = NK * ROW;                              // bytes of a block of keys or values
    constexpr int STAGE = 8 * BLOCK + 8 * KT;                    // a run: keys, values, both scales
    extern __shared__ __align__(128) float smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    __shared__ SingleLine<LINE> line;
    int walker = 0, x = 0, x_end = 1;                            // LINE: this warp's part of the line
    if constexpr (LINE) {
        ST_PDL_TRIGGER();
        walker = blockIdx.x * SG_LINE_WARPS + warp;
        sg_line_begin<KT>(a, line);
        x = (int)min((long long)walker * line.run, (long long)line.total);
        x_end = (int)min((long long)x + line.run, (long long)line.total);
    }
    while (x < x_end) {
    int item, part, i, i_end, stride;                            // part: key head and row block; runs i, i + stride, ... below i_end
    if constexpr (LINE) {
        part = x / line.length;
        const int r = x - part * line.length;
        item = sg_line_find(line, a.n_items, r);
        const int first = line.before[item], n = line.before[item + 1] - first;
        i = r - first;
        i_end = min(n, i + x_end - x);
        stride = 1;
    } else {
        item = blockIdx.x / a.splits;
        part = blockIdx.y;
        i = blockIdx.x % a.splits * W + warp;
        stride = W * a.splits;
        i_end = 1 << 30;
    }
    const int key_head = part / a.row_blocks, head0 = key_head * a.group + (part % a.row_blocks) * R;
    const int rows = min(R, (key_head + 1) * a.group - head0);
    const int token = a.items ? a.items[item] : item, pos = token >= 0 ? __ldg(a.positions + token) : -1;
    const int seq = token >= 0 ? __ldg(a.seq_of_token + token) : 0;
    if (!LINE && pos < 0) {                                      // (the same for all blocks of a cluster)
        if (a.info) ST_PDL_WAIT();                               // this kernel never ends before the one it was let in by
        return;
    }
    const int* bt = a.kv.table + (size_t)__ldg(a.slots + seq) * a.kv.max_pages;
    const SingleSpan span = sg_span(a, item, pos);
    const int lo = span.lo, hi = span.hi;
    if (!LINE && pos >= a.kv.reach && a.kv.status) *a.kv.status = 1;
    const int i0 = i;
    // offset of this lane's word w in a key row: pieces of 16 bytes per lane while the row lasts, then 8, then 4
    auto key_byte = [&](int w) -> int {
        constexpr int full = KW / 4 * 4, two = KW % 4 / 2 * 2;
        if (w < full) return (w / 4) * 64 + t * 16 + (w % 4) * 4;
        if (w < full + two) return full * 16 + t * 8 + (w - full) * 4;
        return (full + two) * 16 + t * 4;
    };
    const int base0 = lo & ~7, runs = min(i_end, hi > lo ? (hi - base0 + KT - 1) / KT : 0);
    // A run's keys are four aligned blocks of NK, each within a page.  Lane (g, t) looks up block t, two runs ahead (ask), and
    // turns the page into a row of the pool one run ahead (resolve); its rows' keys are in block g / 2, whose row lane g / 2 has.
    constexpr uint32_t NONE = 0xffffffffu;
    const uint32_t to_values = (uint32_t)a.kv.nkv * a.kv.page_size;
    int page = -1, off = 0;
    auto ask = [&](int i) {
        const int key = base0 + i * KT + t * NK;
        page = -1;
        if (key < hi) {
            const int index = a.kv.page_index(key);
            off = a.kv.offset(key, index);
            if (index < a.kv.max_pages) page = __ldg(bt + index);
        }
    };
    auto resolve = [&](int i) -> uint32_t {
        const int key = base0 + i * KT + t * NK;
        if (i >= runs || key >= hi) return NONE;
        if ((unsigned)page >= (unsigned)a.kv.num_pages) {
            if (key + NK > lo && a.kv.status) *a.kv.status = 1;
            return NONE;
        }
        return a.kv.row0(page, 0, key_head) + off;
    };
    // ---- a run's copies: lane t has block t's row of the pool.  A lane's places are the same in every block but for bits of the address
    // that the block's number turns over (the stages and blocks lie on multiples of 128 bytes).
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (STAGES * STAGE);
    constexpr int CHUNKS = (BLOCK + 511) / 512;
    const unsigned char* const keys_of = a.kv.pool + lane * 16;
    const unsigned char* const values_of = keys_of + (size_t)to_values * ROW;
    const int w_lane = lane / (NK / 4), c_lane = lane % (NK / 4);    // NK / 4 pieces of the keys' scales, as many of the values'
    const float* const scales_of = a.kv.scales + (HALF && lane < NK / 2 ? w_lane * to_values + c_lane * 4 : 0u);
    uint32_t key_to[CHUNKS], value_to[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int b = c * 512 + lane * 16, k = b / ROW, e = b % ROW;
        key_to[c] = sg_key_at<ROW>(k, e);
        value_to[c] = 4 * BLOCK + sg_value_at<ROW, NK>(0, k, e);
    }
    const uint32_t scale_to = 8 * BLOCK + (w_lane * KT + c_lane * 4) * 4;
    auto copy = [&](uint32_t at, uint32_t stage) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const uint32_t r = __shfl_sync(0xffffffffu, at, b);
            const bool ok = r != NONE;
            const uint32_t row = ok ? r : 0u;
            constexpr uint32_t turn = ROW == 64 ? 1 : 0;             // block b's values: (b & 1) << 6 | (b >> 1) << 5, or b << 5
            const uint32_t bits = turn ? (uint32_t)((b & 1) << 6 | (b >> 1) << 5) : ROW % 128 == 0 ? (uint32_t)(b << 5) : 0u;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                if (c * 512 + lane * 16 >= BLOCK) continue;
                sg_copy16(stage + key_to[c] + b * BLOCK, keys_of + (size_t)row * ROW + c * 512, ok);
                sg_copy16(((stage + value_to[c]) ^ bits) + b * BLOCK, values_of + (size_t)row * ROW + c * 512, ok);
            }
            if (HALF && lane < NK / 2) sg_copy16(stage + scale_to + b * NK * 4, scales_of + row, ok);
        }
    };
    // an eighth of a value row: of every 128 (8-bit forms) or 64 dimensions 16 or 8 neighbours, of 32 four, of 16 two
    constexpr int V16 = B == 1 ? D / 128 : 0, V8 = (D - 128 * V16) / 64, V4 = D % 64 / 32, V2 = D % 32 / 16;
    auto value_dim = [&](int n, int i) -> int {                 // the i-th dimension that lanes of g = n read
        if (i < 16 * V16) return n * 16 + i;
        if (i < 16 * V16 + 8 * V8) return 128 * V16 + ((i - 16 * V16) >> 3) * 64 + n * 8 + (i & 7);
        if (i < 16 * V16 + 8 * V8 + 4 * V4) return 128 * V16 + 64 * V8 + n * 4 + (i - 16 * V16 - 8 * V8);
        return 128 * V16 + 64 * V8 + 32 * V4 + n * 2 + (i - 16 * V16 - 8 * V8 - 4 * V4);
    };
    auto sees_all = [&](uint32_t at, int key) -> bool { return __all_sync(0xffffffffu, at != NONE && key >= lo && key + NK <= hi); };

    // the first runs' copies leave before the query's loads
    uint32_t at[STAGES];                                      // block t's row of runs i, i + stride, ...
    ask(i);
#pragma unroll
    for (int j = 0; j + 1 < STAGES; ++j) {
        at[j] = resolve(i + j * stride);
        ask(i + (j + 1) * stride);
        copy(at[j], ring + j * STAGE);
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    }

    // ---- the query's fragments: column g is head g (TWO: head g % 4, its second number from column 4 on)
    uint32_t qb[NS][2];
    float fac[2] = {a.scale_log2, a.scale_log2};                 // of the heads of columns 2 t and 2 t + 1
    {
        const int r = TWO ? g & 3 : g;
        const bool ok = r < rows;
        const QT* q = (const QT*)a.q + ((size_t)token * a.nh + head0 + (ok ? r : 0)) * D;
        float v[NS][4];
        uint32_t amax = 0;
#pragma unroll
        for (int x = 0; x < NS; ++x)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // element 4 x + k of the lane's quarter row: a word holds 4 / B of them
                const int e = 4 * x + k, dim = key_byte(e * B / 4) / B + e % (4 / B);
                v[x][k] = ok ? to_f32(q[dim]) : 0.f;
                amax = max(amax, __float_as_uint(v[x][k]) & 0x7fffffffu);
            }
        float mul = 1.f;
        if (HALF) {
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int ex = min(max((int)(amax >> 23) - 127, -100), 127);
            mul = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
            const float f = ldexpf(a.scale_log2, ex - 14);
            fac[0] = __shfl_sync(0xffffffffu, f, 8 * t);
            fac[1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
        }
#pragma unroll
        for (int x = 0; x < NS; ++x)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const float y = v[x][2 * p] * mul, z = v[x][2 * p + 1] * mul;
                uint32_t w = sg_pack<HALF>(y, z);
                if (FLOATQ) {
                    const float2 f = sg_unpack<HALF>(w);
                    if (g >= 4) w = sg_pack<HALF>(y - f.x, z - f.y);
                }
                qb[x][p] = w;
            }
    }
    float ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, acc[NT / 2][4];
#pragma unroll
    for (int j = 0; j < NT / 2; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[j][k] = 0.f;

    uint32_t now = 0;                                            // the stage of run i
    for (; i < runs; i += stride) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory");
        __syncwarp();                                            // run i has landed, and every lane is done with the run before it
        const uint32_t stage = ring + now * STAGE;
        {
            const uint32_t last = now == 0 ? STAGES - 1 : now - 1;
            at[STAGES - 1] = resolve(i + (STAGES - 1) * stride);
            ask(i + STAGES * stride);
            copy(at[STAGES - 1], ring + last * STAGE);
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        }
        const uint32_t at_k = __shfl_sync(0xffffffffu, at[0], g >> 1);
        const bool all = sees_all(at[0], base0 + i * KT + t * NK);
        // ---- scores: rows g and g + 8 of product m are keys 4 m + g % 2 and 4 m + g % 2 + 2 of block g / 2
        float s[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            uint32_t kw[2][KW];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                constexpr int full = KW / 4 * 4, two = KW % 4 / 2 * 2;
                const int row = (g >> 1) * NK + 4 * m + 2 * h + (g & 1);
#pragma unroll
                for (int w = 0; w < full; w += 4) sg_load<4>(stage + sg_key_at<ROW>(row, key_byte(w)), kw[h] + w);
                if constexpr (two > 0) sg_load<2>(stage + sg_key_at<ROW>(row, key_byte(full)), kw[h] + full);
                if constexpr (full + two < KW) sg_load<1>(stage + sg_key_at<ROW>(row, key_byte(full + two)), kw[h] + full + two);
            }
#pragma unroll
            for (int x = 0; x < NS; ++x) {
                uint32_t f[4];
                if constexpr (HALF) {
                    c8_halves<FORM>(kw[0][x], f[0], f[2]);
                    c8_halves<FORM>(kw[1][x], f[1], f[3]);
                } else {
                    f[0] = kw[0][2 * x]; f[2] = kw[0][2 * x + 1];
                    f[1] = kw[1][2 * x]; f[3] = kw[1][2 * x + 1];
                }
                if (x == 0) sg_mma<HALF, false>(s[m], f, qb[x][0], qb[x][1]);
                else sg_mma<HALF, true>(s[m], f, qb[x][0], qb[x][1]);
            }
        }
        float ks[2 * MT], vs[2 * MT];                            // of the keys of this lane's scores
        if (HALF) {
#pragma unroll
            for (int j = 0; j < 2 * MT; ++j) {
                const uint32_t p = stage + 8 * BLOCK + ((g >> 1) * NK + (g & 1) + 2 * j) * 4;
                asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(ks[j]) : "r"(p));
                asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(vs[j]) : "r"(p + KT * 4));
            }
        }
        // ---- softmax's numbers: s[m][c], s[m][2 + c] are column 2 t + c at keys 2 m and 2 m + 1 of ks and vs
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (FLOATQ) s[m][k] += __shfl_xor_sync(0xffffffffu, s[m][k], 2);
                if (HALF) s[m][k] *= ks[2 * m + (k >> 1)];
            }
        if (!all) {
            const int key = base0 + i * KT + (g >> 1) * NK + (g & 1);
#pragma unroll
            for (int j = 0; j < 2 * MT; ++j)
                if (at_k == NONE || key + 2 * j < lo || key + 2 * j >= hi) {
                    vs[j] = 0.f;                                 // (a row that is not finite has the scale NaN)
                    s[j >> 1][2 * (j & 1)] = s[j >> 1][2 * (j & 1) + 1] = -INFINITY;
                }
        }
        float lead = 0.f;                                        // log2 of the largest value scale, rounded up
        if (HALF) {
            float vmax = vs[0];
#pragma unroll
            for (int j = 1; j < 2 * MT; ++j) vmax = fmaxf(vmax, vs[j]);
            lead = (float)max((int)(__float_as_uint(vmax) >> 23) - 126, -90);
        }
        float corr[2];
        bool move = false;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(s[0][c], s[0][2 + c]);
            if constexpr (MT == 2) mx = fmaxf(mx, fmaxf(s[MT - 1][c], s[MT - 1][2 + c]));
            mx = fmaf(mx, fac[c], lead);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            corr[c] = 1.f;
            if (mx > ref[c] + 15.f) {
                const float r = mx - 11.f;
                corr[c] = ar_exp2(ref[c] - r);                   // 0 from "no key yet"
                ref[c] = r;
                move = true;
            }
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                sum[c] *= corr[c];
#pragma unroll
                for (int j = 0; j < NT / 2; ++j) { acc[j][c] *= corr[c]; acc[j][2 + c] *= corr[c]; }
            }
        }
        uint32_t pb[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {                        // keys of rows g, of rows g + 8
                float z[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float neg = ref[c] == -INFINITY ? 0.f : -ref[c];
                    const float p = ar_exp2(fmaf(s[m][2 * h + c], fac[c], neg));
                    sum[c] += p;
                    z[c] = HALF ? p * vs[2 * m + h] : p;
                }
                uint32_t w = sg_pack<HALF>(z[0], z[1]);
                if (TWO) {
                    const float2 f = sg_unpack<HALF>(w);
                    if (t >= 2) w = sg_pack<HALF>(z[0] - f.x, z[1] - f.y);
                }
                pb[m][h] = sg_transpose(w);
            }
        // ---- values times weights: rows g and g + 8 of product j are this lane's dimensions 2 j and 2 j + 1
        uint32_t vw[NK][VW];
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const uint32_t v = stage + 4 * BLOCK;
            if constexpr (V16) sg_load<4>(v + sg_value_at<ROW, NK>(t, k, g * 16), vw[k]);
#pragma unroll
            for (int c = 0; c < V8; ++c) {
                if constexpr (B == 1) sg_load<2>(v + sg_value_at<ROW, NK>(t, k, (V16 * 128 + c * 64 + g * 8) & ~15) + (g & 1) * 8, vw[k] + 4 * V16 + 2 * c);
                else sg_load<4>(v + sg_value_at<ROW, NK>(t, k, c * 128 + g * 16), vw[k] + 4 * c);
            }
            if constexpr (V4) {
                constexpr int from = V8 * 64 * B;
                const int b = from + g * 4 * B;
                if constexpr (B == 1) sg_load<1>(v + sg_value_at<ROW, NK>(t, k, b & ~15) + (b & 15), vw[k] + 2 * V8);
                else sg_load<2>(v + sg_value_at<ROW, NK>(t, k, b & ~15) + (b & 15), vw[k] + 4 * V8);
            }
            if constexpr (V2) {
                constexpr int from = (V8 * 64 + V4 * 32) * B;
                const int b = from + g * 2 * B;
                if constexpr (B == 1) vw[k][VW - 1] = sg_load2(v + sg_value_at<ROW, NK>(t, k, b & ~15) + (b & 15));
                else sg_load<1>(v + sg_value_at<ROW, NK>(t, k, b & ~15) + (b & 15), vw[k] + VW - 1);
            }
        }
        if (!all) {
            // hidden rows may hold anything: zeros in their place
            const int key = base0 + i * KT + t * NK;
#pragma unroll
            for (int k = 0; k < NK; ++k)
                if (key + k < lo || key + k >= hi) {
#pragma unroll
                    for (int w = 0; w < VW; ++w) vw[k][w] = 0u;
                }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
            constexpr int PER = 4 / B;                           // dimensions of a word
            uint32_t b[MT][2][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t x = vw[4 * m + 2 * h][w], y = vw[4 * m + 2 * h + 1][w];
                    if constexpr (HALF) c8_pairs<FORM>(x, y, b[m][h]);
                    else { b[m][h][0] = __byte_perm(x, y, 0x5410); b[m][h][1] = __byte_perm(x, y, 0x7632); }
                }
#pragma unroll
            for (int c = 0; c < PER; c += 2) {
                const int j = (w * PER + c) / 2;
                if (2 * j < NT) {
                    float o[4];
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint32_t f[4] = {b[m][0][c], b[m][0][c + 1], b[m][1][c], b[m][1][c + 1]};
                        if (!FLOATQ) sg_mma<HALF, true>(acc[j], f, pb[m][0], pb[m][1]);
                        else if (m == 0) sg_mma<HALF, false>(o, f, pb[m][0], pb[m][1]);
                        else sg_mma<HALF, true>(o, f, pb[m][0], pb[m][1]);
                    }
                    if (FLOATQ) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[j][k] += o[k];
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j + 1 < STAGES; ++j) at[j] = at[j + 1];
        now = now + 1 == STAGES ? 0 : now + 1;
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncwarp();                                                // the ring is free
    if constexpr (!LINE) __syncthreads();                        // the parts lie where the rings were
    // ---- the columns' sums
    const int unit = LINE ? part * a.n_items + item : 0;
    const bool whole = LINE && !a.info && i0 == 0 && i_end == line.before[item + 1] - line.before[item];
    const size_t slot = LINE ? (size_t)(unit + walker) * R : 0;
    float* s_ref = smem;
    float* s_sum = s_ref + W * R;
    float* s_acc = s_sum + W * R;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        float l = sum[c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const int r = 2 * t + c;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (g == 0 && r < R) {
            if constexpr (LINE) {
                if (!whole) { a.line.r[slot + r] = ref[c]; a.line.l[slot + r] = l; }
            } else {
                s_ref[warp * R + r] = ref[c];
                s_sum[warp * R + r] = l;
            }
        }
#pragma unroll
        for (int j = 0; j < NT / 2; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float o = acc[j][2 * h + c];
                if (TWO) o += __shfl_xor_sync(0xffffffffu, o, 2);
                const int e = value_dim(g, 2 * j + h);
                if (r < rows) {
                    if constexpr (!LINE) s_acc[((size_t)warp * R + r) * D + e] = o;
                    else if (whole) ((QT*)a.out)[((size_t)token * a.nh + head0 + r) * D + e] = from_f32<QT>(o * inv);
                    else a.line.o[(slot + r) * D + e] = o;
                }
            }
    }
    if constexpr (!LINE) {
        sg_finish<QT>(a, smem, W, R, rows, D, token, pos, item, head0, key_head);
        return;
    }
    if (i0 == 0 && lane == 0) {
        a.span[2 * unit] = walker;
        a.span[2 * unit + 1] = (x + line.before[item + 1] - line.before[item] - 1) / line.run;
    }
    x += i_end - i0;
    }
    if (LINE && a.info) ST_PDL_WAIT();                           // this kernel never ends before the one it was let in by
}

// Blocks, warps and the cluster: n_pairs = items x row blocks of all key heads, each over up to max_keys keys.
struct SingleShape { int splits, warps; };
SingleShape sg_shape(long long n_pairs, int max_keys, int keys_per_run);

template <typename K>
static inline int sg_launch(const char* tag, K kernel, const SingleArgs& a, dim3 grid, int warps, size_t smem, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
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

template <int FORM, typename QT, int D, bool TWO>
static int sg_run(SingleArgs a, int max_keys, cudaStream_t s) {
    constexpr int R = TWO ? 4 : 8, ROW = D * c8_bytes(FORM), KT = sg_run_keys(ROW);
    a.row_blocks = (a.group + R - 1) / R;
    const int grid_y = a.row_blocks * a.kv.nkv;
    constexpr size_t RING = sg_stages(ROW) * (2 * KT * ROW + 8 * KT);       // bytes per warp
    if (a.walkers) {
        const size_t smem = SG_LINE_WARPS * RING;
        AR_ALLOW_SMEM((attention_single8_kernel<FORM, QT, D, TWO, true>), smem);
        const int rc = sg_launch("single8", attention_single8_kernel<FORM, QT, D, TWO, true>, a, dim3(a.walkers / SG_LINE_WARPS), SG_LINE_WARPS, smem, s);
        if (rc) return rc;
        // few units have many parts each (110 for four long caches: 35.4 us in all with 512 threads, 36.9 with 256), many units two or three
        const int units = a.n_items * grid_y;
        return st_launch_pdl("single8_join", attention_single8_join_kernel<QT, KT>, dim3(units, a.group < R ? a.group : R),
                             dim3(units < a.walkers / 8 ? SG_JOIN : 64), 0, s, a, R);
    }
    SingleShape shape = sg_shape((long long)a.n_items * grid_y, max_keys, KT);
    while (shape.warps * RING > SG_SMEM) shape.warps /= 2;
    a.splits = shape.splits;
    static_assert((size_t)SG_MAX_WARPS * R * (D + 2) * 4 <= SG_SMEM, "");
    const size_t parts = (size_t)shape.warps * R * (D + 2) * 4, rings = shape.warps * RING, smem = parts > rings ? parts : rings;
    AR_ALLOW_SMEM((attention_single8_kernel<FORM, QT, D, TWO, false>), SG_SMEM);
    return sg_launch("single8", attention_single8_kernel<FORM, QT, D, TWO, false>, a, dim3((unsigned)a.n_items * a.splits, grid_y), shape.warps,
                     smem, s);
}
template <int FORM, typename QT, bool TWO> static int sg_run(const SingleArgs& a, int max_keys, cudaStream_t s) {
    if (a.d == 32) return sg_run<FORM, QT, 32, TWO>(a, max_keys, s);
    if (a.d == 64) return sg_run<FORM, QT, 64, TWO>(a, max_keys, s);
    if (a.d == 80) return sg_run<FORM, QT, 80, TWO>(a, max_keys, s);
    if (a.d == 96) return sg_run<FORM, QT, 96, TWO>(a, max_keys, s);
    if (a.d == 128) return sg_run<FORM, QT, 128, TWO>(a, max_keys, s);
    return ST_ERR_BAD_SIZE;
}

// How a call is dealt out as one line, walkers 0 if it is not.  The line costs a second launch and parts through memory, and pays from
// two runs a warp on.  Blocks against the line, in us, 32 heads of 64 in int8: 5.4 / 8.9 at 0.4 runs a warp, 9.6 / 11.6 at 1.7,
// 14.9 / 13.0 at 2.6, 18.3 / 16.1 at 3.5, 26.6 / 24.4 at 10, 63.4 / 61.7 at 41; 4 heads of 128 behind long caches: 18.4 / 16.9
// at 1.1, 38.3 / 25.8 at 4.5, 57.2 / 35.7 at 9.  Requests of one length whose blocks fill the device in whole turns lose by it: 32 of 1000
// keys each (32 heads of 64, int8, 14 runs a warp) 32.6 / 36.4, 64 of them 58.3 / 59.7.  Lengths are in device memory; the host
// knows about the longest only, and gives this up for 16 of 1000 (25.1 / 24.2), 64 of 250 (28.5 / 25.8) and all unequal ones.
struct LineShape { int walkers, R; long long slots; };
static inline LineShape sg_line_shape(int n_items, int group, int nkv, int d, int max_keys, long long reach, bool float_q, int form) {
    LineShape s{0, float_q || (form == C8_BF16 && group <= 4) ? 4 : 8, 0};
    const int row = d * c8_bytes(form), kt = sg_run_keys(row), walkers = st_sm_count() * sg_line_blocks(row) * SG_LINE_WARPS;
    const long long parts = (long long)n_items * nkv * ((group + s.R - 1) / s.R), runs = parts * ((max_keys + kt - 1) / kt);
    // (the device counts the line's runs, of up to `reach` keys a token, in 32 bits)
    if (n_items > SG_LINE_ITEMS || runs < 2ll * walkers || parts * (reach / kt + 2) >= (1 << 30)) return s;
    s.walkers = walkers;
    s.slots = parts + walkers;
    return s;
}

int sg_int8(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s);
int sg_e4m3(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s);
int sg_bf16(const SingleArgs& a, int max_keys, cudaStream_t s);
// the kernels in float arithmetic, for every size (attention_rows_any.cuh)
int aa_single_int8(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s);
int aa_single_e4m3(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s);
int aa_single_wide(const SingleArgs& a, bool float_q, int max_keys, cudaStream_t s);
