// What the attention kernels over 8-bit caches and over shared prefixes have in common: the tiles of query rows a plan names,
// how their work is dealt out, and the parts of a row's softmax that different blocks leave for one another.
//
// A row is one (token, query head).  A tile holds the rows of up to 128 / g tokens, for one key head, g = query heads per key
// head: row r is head r % g of the group of token r / g.  The tile's keys [key_lo, key_hi) are walked in chunks of AR_CHUNK.
// All chunks of all (tile, key head) pairs ("units"), one unit's behind the other's, each unit with AR_UNIT places in front for what its
// begin and end cost (without them the walkers of a prompt's first, short units were the last by a factor of two), form one line
// of `total` places which is cut
// into runs of `run` places, one per walker (a block, or one of a block's two groups): every walker gets the same work however
// unequal the tiles are, and a unit that a cut goes through is put together from parts.  Where results leave directly, a walker leaves
// two parts at most: what it began with, of a unit that a cut in front of it went through, has slot 2 c of walker c, what it ended
// with, the begin of a unit, slot 2 c + 1.  Of shared keys every piece is a part: that of unit u and walker c has slot u + c (a new slot
// begins with every unit and with every run, so no two parts share one).
//
// A part of a row is (R, l, O): p_j = 2^(s_j - R), s in units of log2, l = sum p_j, O = sum p_j v_j, all float; R is a number near
// the largest s_j (the exact maximum is not needed: only the common factor).  Parts are joined by 2^(R - max R).
#pragma once
#include <atomic>

#include "cache8.cuh"

#define AR_ROWS 128
#define AR_CHUNK 64
#define AR_UNIT 3                 // what a unit's begin and end cost, in chunks
#define AR_LOG2E 1.4426950408889634f

// a tile of a plan: six numbers in the plan's array
struct RowTile { int first, n_tok, seq, key_lo, key_hi, start; };   // start: the line's place where key head 0's share begins

struct RowPlan {
    const int* tiles;        // [n_tiles][6]
    const int* items;        // tokens in the tiles' order, or null: tile tokens are first, first + 1, ...
    int n_tiles, total, ctas, run;
    int nh, nkv, group;      // group = nh / nkv
};
// where parts lie: per slot AR_ROWS rows (R, l) and AR_ROWS x d of O
struct RowParts {
    float* r;
    float* l;
    float* o;
};
__host__ __device__ inline size_t ar_part_floats(int d) { return (size_t)AR_ROWS * (2 + d); }

// what the kernels of tiles get
struct RowArgs {
    const void* q;
    void* out;
    long long q_stride;              // elements between the query rows of neighbouring tokens
    PagedKV kv;
    RowPlan plan;
    RowParts parts;
    const int* positions;
    const int* seq_of_token;
    const int* slots;
    int d, window;
    int direct;                      // a unit that one block has wholly goes to `out`; else every piece to its slot
    float scale_log2;
};

__device__ __forceinline__ RowTile ar_tile(const RowPlan& p, int i) {
    const int* t = p.tiles + 6 * i;
    return RowTile{__ldg(t), __ldg(t + 1), __ldg(t + 2), __ldg(t + 3), __ldg(t + 4), __ldg(t + 5)};
}
__device__ __forceinline__ int ar_chunks(const RowTile& t) {
    return t.key_hi > t.key_lo ? (t.key_hi - (t.key_lo & ~(AR_CHUNK - 1)) + AR_CHUNK - 1) / AR_CHUNK : 0;
}
__device__ __forceinline__ int ar_places(int chunks) { return chunks > 0 ? chunks + AR_UNIT : 0; }      // of a unit in the line

// Token i of a tile, and its position (-1: padding, whose request may be any number).
struct RowMember { int token, pos; };
__device__ __forceinline__ RowMember ar_member(const RowArgs& a, const RowTile& t, int i) {
    RowMember m{-1, -1};
    if (i < t.n_tok) {
        m.token = a.plan.items ? __ldg(a.plan.items + t.first + i) : t.first + i;
        m.pos = __ldg(a.positions + m.token);
    }
    return m;
}
__device__ __forceinline__ int ar_low(const RowArgs& a, int pos) { return a.window > 0 ? pos - a.window + 1 : 0; }   // the first key seen from pos

// The block table's row by which keys lo .. hi of a tile are found: its request's for all keys; of a tile of shared keys that of the first
// member that is not padding, for the keys that this one sees.  Of other keys it may have none, be it that it stands before them or
// that its window has left them behind: these belong to the first member that sees them (ar_first), and to nobody if none does.
struct RowTable { const int* row; int lo, hi; };
__device__ __forceinline__ const int* ar_row(const RowArgs& a, int seq) { return a.kv.table + (size_t)__ldg(a.slots + seq) * a.kv.max_pages; }
template <bool SHARED> __device__ __forceinline__ RowTable ar_table(const RowArgs& a, const RowTile& t) {        // by a whole warp
    if (!SHARED) return RowTable{ar_row(a, t.seq), 0, 0x7fffffff};
    for (int i = 0; i < t.n_tok; i += 32) {
        const RowMember m = ar_member(a, t, i + (threadIdx.x & 31));
        const int seq = m.token >= 0 ? __ldg(a.seq_of_token + m.token) : 0;      // beside the positions, though one member's is used
        const uint32_t live = __ballot_sync(0xffffffffu, m.pos >= 0);
        if (!live) continue;
        const int src = __ffs(live) - 1, pos = __shfl_sync(0xffffffffu, m.pos, src);
        return RowTable{ar_row(a, __shfl_sync(0xffffffffu, seq, src)), ar_low(a, pos), pos};
    }
    return RowTable{nullptr, 1, 0};
}
// The first token of a tile that sees `key`, or -1: by a whole warp, a key per lane that asks.
__device__ __forceinline__ int ar_first(const RowArgs& a, const RowTile& t, int key, bool asks) {
    int found = -1;
    for (int i = 0; i < t.n_tok && __any_sync(0xffffffffu, asks && found < 0); i += 32) {
        const RowMember m = ar_member(a, t, i + (threadIdx.x & 31));
        const int low = m.pos >= 0 ? ar_low(a, m.pos) : 0x7fffffff;
        // most keys that the tile's first member does not see nobody sees: they lie outside of all members' keys
        const int last = __reduce_max_sync(0xffffffffu, m.pos), first = __reduce_min_sync(0xffffffffu, low);
        if (!__any_sync(0xffffffffu, asks && found < 0 && key <= last && key >= first)) continue;
        const int n = min(32, t.n_tok - i);
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            const int token = __shfl_sync(0xffffffffu, m.token, j), pos = __shfl_sync(0xffffffffu, m.pos, j);
            const int least = __shfl_sync(0xffffffffu, low, j);
            if (asks && found < 0 && key <= pos && key >= least) found = token;
        }
    }
    return found;
}
// Whether a token of a tile sees `key`: asked where a key of a portion has no page, which padding behind the portion need not have.
__device__ __forceinline__ bool ar_needed(const RowArgs& a, const RowTile& t, int key) {
    bool seen = false;
#pragma unroll 1
    for (int i = 0; i < t.n_tok; ++i) {
        const int pos = __ldg(a.positions + t.first + i);
        seen |= key <= pos && key >= ar_low(a, pos);
    }
    return seen;
}
// The block table's row by which a lane's key is found; null: the key is not asked for.  By a whole warp.
template <bool SHARED>
__device__ __forceinline__ const int* ar_row_of(const RowArgs& a, const RowTile& t, const RowTable& table, int key, bool in_tile) {
    if (!SHARED) return in_tile ? table.row : nullptr;
    const bool there = in_tile && key >= table.lo && key <= table.hi, other = in_tile && !there;
    const int* row = there ? table.row : nullptr;
    if (__any_sync(0xffffffffu, other)) {
        const int token = ar_first(a, t, key, other);
        if (token >= 0) row = ar_row(a, __ldg(a.seq_of_token + token));
    }
    return row;
}

// A walker's way along its run: pieces of one (tile, key head) pair.  A walker behind the line's end has none.
struct RowPiece {
    RowTile t;
    int tile, head;          // head: key head
    int unit, chunk0, chunks;   // chunks of the unit done here, from chunk0 on
    bool whole;              // this piece is all of its unit
};
struct RowWalk {
    int at, end, tile;
    RowTile t;
    // by a whole warp
    __device__ __forceinline__ void begin(const RowPlan& p, int c) {
        at = min(c * p.run, p.total);
        end = min(at + p.run, p.total);
        // the last tile that starts at or before `at` (tiles without chunks start where the next one does), by 32 at a time
        int lo = 0, n = p.n_tiles;
        while (n > 1) {
            const int step = (n + 31) / 32, i = lo + (int)(threadIdx.x & 31) * step;
            const bool before = i < lo + n && __ldg(p.tiles + 6 * i + 5) <= at;
            const uint32_t set = __ballot_sync(0xffffffffu, before);
            const int k = set ? 31 - __clz(set) : 0;
            n = min(step, n - k * step);
            lo += k * step;
        }
        tile = lo;
        t = ar_tile(p, tile);
    }
    __device__ __forceinline__ bool next(const RowPlan& p, RowPiece& out) {
        if (at >= end) return false;
        int n = ar_chunks(t);
        while (at >= t.start + ar_places(n) * p.nkv) {
            if (++tile >= p.n_tiles) return false;
            t = ar_tile(p, tile);
            n = ar_chunks(t);
        }
        const int in = at - t.start, head = in / ar_places(n);
        int c = in - head * ar_places(n);
        if (c < AR_UNIT) {                               // the unit's own places
            at += AR_UNIT - c;
            c = AR_UNIT;
            if (at >= end) return false;
        }
        out.t = t;
        out.tile = tile;
        out.head = head;
        out.unit = tile * p.nkv + head;
        out.chunk0 = c - AR_UNIT;
        out.chunks = min(n - out.chunk0, end - at);
        out.whole = out.chunks == n;
        at += out.chunks;
        return true;
    }
};
// the walkers of unit (tile t, key head) with n > 0 chunks: c0 to c1
__device__ __forceinline__ void ar_walkers(const RowPlan& p, const RowTile& t, int head, int n, int& c0, int& c1) {
    const int x0 = t.start + head * ar_places(n) + AR_UNIT;
    c0 = x0 / p.run;
    c1 = (x0 + n - 1) / p.run;
}

__device__ __forceinline__ int ar_slot(const RowArgs& a, const RowPiece& p, int walker) {      // of a piece that is not direct
    return a.direct ? 2 * walker + (p.chunk0 == 0) : p.unit + walker;
}

__device__ __forceinline__ float ar_exp2(float x) {      // 2 ulp, exp2(-inf) = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// the weight of a part with reference r beside the largest reference m (none: -inf)
__device__ __forceinline__ float ar_weight(float r, float m) { return r == -INFINITY ? 0.f : ar_exp2(r - m); }

static inline int ar_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? dev : 0;
}
// Dynamic shared memory above 48 KB is asked for once per kernel and device, `most` that any call of the kernel takes: two threads whose first
// calls meet then set the same number, and neither launches with more than the other has left allowed.
#define AR_ALLOW_SMEM(kernel, most)                                                                                      \
    do {                                                                                                                 \
        static std::atomic<bool> allowed[64];                                                                            \
        std::atomic<bool>& have = allowed[ar_device()];                                                                  \
        if ((size_t)(most) > 48 * 1024 && !have) {                                                                       \
            const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(most)); \
            if (err != cudaSuccess) { cudaGetLastError(); return (int)err; }                                             \
            have = true;                                                                                                 \
        }                                                                                                                \
    } while (0)

// tiles on the tensor cores (attention_rows_tc.cu): bfloat16 queries, 8-bit and bfloat16 caches, head sizes that are multiples of 16
// up to 128
int ar_rows_tc(const RowArgs& a, int form, cudaStream_t s);
// tiles in float arithmetic, every size (attention_rows_any.cuh)
int aa_rows_int8(const RowArgs& a, bool float_q, int max_rows, cudaStream_t s);
int aa_rows_e4m3(const RowArgs& a, bool float_q, int max_rows, cudaStream_t s);
int aa_rows_wide(const RowArgs& a, bool float_q, int max_rows, cudaStream_t s);
