// Attention over 8-bit caches and shared prefixes: the kernel that joins the parts of a unit, and the entry points, which choose between
// the tensor-core kernels (attention_rows_tc.cu, attention_single8.cuh) and those in float arithmetic (attention_rows_any.cuh).
#include "attention_single8.cuh"

// ---- joining the parts of units that a cut goes through ------------------------------------------------------------
// Blocks (c, .) look at the cut in front of run c, and join the unit there if it is the first cut through it.  Bound by latency: two to
// a few parts per row, four dimensions per thread (9 us for 2000 tokens of 32 heads of 64, 13 for 1000 behind 1500 keys, 32 heads of 128).
template <typename QT>
__global__ void __launch_bounds__(256) attention_rows_join_kernel(const RowArgs a) {
    const RowPlan& p = a.plan;
    const int x = blockIdx.x * p.run, d = a.d, g = p.group;
    RowWalk w;
    w.begin(p, blockIdx.x);
    RowPiece pc;
    int c0 = -1, c1 = -1;
    if (x > 0 && x < p.total && w.next(p, pc) && pc.chunk0 > 0)     // else the run begins with a unit of its own
        ar_walkers(p, pc.t, pc.head, ar_chunks(pc.t), c0, c1);
    ST_PDL_WAIT();                                                  // by all blocks: what follows this kernel follows the tiles' too
    if (c0 < 0 || c0 != (int)blockIdx.x - 1) return;
    const int pieces = (d + 3) / 4, total = pc.t.n_tok * g * pieces, n = c1 - c0 + 1;
    const bool vec = d % 4 == 0, wide = vec && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
    for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < total; i += gridDim.y * blockDim.x) {
        const int r = i / pieces, e = (i - r * pieces) * 4, place = pc.t.first + r / g, token = p.items ? p.items[place] : place;
        const int pos = a.positions[token];
        // two parts at a time, all of their numbers under way together; what was summed before moves to the largest reference so far
        float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < n; k += 2) {
            float ref[2], sum[2], x[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = k + (k + h < n ? h : 0);              // part 0 ended its walker's run, the others began theirs
                const size_t at = (size_t)(2 * (c0 + j) + (j == 0)) * AR_ROWS + r;
                const float* part = a.parts.o + at * d + e;
                ref[h] = __ldcg(a.parts.r + at);
                sum[h] = __ldcg(a.parts.l + at);
                if (vec) {
                    const float4 v = __ldcg(reinterpret_cast<const float4*>(part));
                    x[h][0] = v.x; x[h][1] = v.y; x[h][2] = v.z; x[h][3] = v.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[h][j] = e + j < d ? __ldcg(part + j) : 0.f;
                }
            }
            if (k + 1 >= n) {                                       // there is no second one: the first was read again
                ref[1] = -INFINITY;
                sum[1] = x[1][0] = x[1][1] = x[1][2] = x[1][3] = 0.f;
            }
            const float most = fmaxf(m, fmaxf(ref[0], ref[1]));
            const float f = ar_weight(m, most), f0 = ar_weight(ref[0], most), f1 = ar_weight(ref[1], most);
            m = most;
            l = l * f + (f0 * sum[0] + f1 * sum[1]);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = o[j] * f + (f0 * x[0][j] + f1 * x[1][j]);
        }
        if (pos < 0) continue;
        QT* out = (QT*)a.out + ((size_t)token * p.nh + pc.head * g + r % g) * d + e;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (wide) {
            store4(out, make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (e + j < d) out[j] = from_f32<QT>(o[j] * inv);
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------
// Warps for a (token, key head) and how they are put into blocks and clusters.  Sixteen warps for every SM keep enough loads in
// flight; a pair gets its share of them, though a warp should have two runs of keys at least, in blocks of four warps (more blocks
// than four warps each need share an SM better than large ones), in clusters of up to eight blocks; only where eight
// such blocks are too few, in larger blocks.
SingleShape sg_shape(long long n_pairs, int max_keys, int keys_per_run) {
    const long long runs = (max_keys + keys_per_run - 1) / keys_per_run;
    long long want = (16ll * st_sm_count() + n_pairs - 1) / n_pairs;
    if (want > (runs + 1) / 2) want = (runs + 1) / 2;
    SingleShape s{1, 4};
    if (want <= 1) { s.warps = runs > 1 ? 4 : 1; if (runs <= 2) s.warps = (int)(runs < 1 ? 1 : runs); return s; }
    while (s.splits < 8 && s.splits * s.warps < want) s.splits *= 2;
    while (s.warps < SG_MAX_WARPS && s.splits * s.warps < want) s.warps *= 2;
    return s;
}

static bool ar_types(int act, int form) {
    return form == C8_INT8 || form == C8_E4M3 ? act == 0 || act == 1 : form == C8_BF16 ? act == 1 : form == C8_F32 && act == 0;
}
static bool ar_single_fast(int page_size, int d, int form) {
    return page_size % 8 == 0 && (d == 32 || d == 64 || d == 80 || d == 96 || d == 128) && form != C8_F32;
}
static int ar_single(const SingleArgs& a, int act, int form, int max_keys, cudaStream_t s) {
    if (ar_single_fast(a.kv.page_size, a.d, form)) {
        if (form == C8_INT8) return sg_int8(a, act == 0, max_keys, s);
        if (form == C8_E4M3) return sg_e4m3(a, act == 0, max_keys, s);
        return sg_bf16(a, max_keys, s);
    }
    if (form == C8_INT8) return aa_single_int8(a, act == 0, max_keys, s);
    if (form == C8_E4M3) return aa_single_e4m3(a, act == 0, max_keys, s);
    return aa_single_wide(a, act == 0, max_keys, s);
}
static bool ar_tc(const RowArgs& a, int act, int form) {
    return act == 1 && form != C8_F32 && a.d % 16 == 0 && a.d <= 128 && aligned16(a.q) && aligned16(a.out) && a.q_stride % 8 == 0;
}
static int ar_rows(RowArgs a, int act, int form, int max_rows, cudaStream_t s) {
    if (ar_tc(a, act, form)) return ar_rows_tc(a, form, s);
    if (form == C8_INT8) return aa_rows_int8(a, act == 0, max_rows, s);
    if (form == C8_E4M3) return aa_rows_e4m3(a, act == 0, max_rows, s);
    return aa_rows_wide(a, act == 0, max_rows, s);
}

// The runs a plan's line is cut into: as many as are walked at the same time, two per SM by the tensor-core kernel, one by every
// block of the float kernel.  No kernel has more walkers for a head size than the float kernel.
static int ar_walkers_most(int d) { return st_sm_count() * (d <= 64 ? 3 : d <= 128 ? 2 : 1); }
static void ar_deal(RowArgs& a, int act, int form) {
    const int most = ar_tc(a, act, form) ? 2 * st_sm_count() : ar_walkers_most(a.d);
    a.plan.run = a.plan.total > most ? (a.plan.total + most - 1) / most : 1;
    a.plan.ctas = (a.plan.total + a.plan.run - 1) / a.plan.run;
}
static RowParts ar_parts(float* scratch, long long slots) {
    return RowParts{scratch, scratch + slots * AR_ROWS, scratch + 2 * slots * AR_ROWS};
}

struct RowCall {            // what the entry points take in common, as the caller lays it out
    const void* q;
    void* out;
    const void* pool;
    const float* scales;
    const int* table;
    const int* positions;
    const int* seq_of_token;
    const int* slots;
    const int* items;
    const int* tiles;
    const int* info;
    float* scratch;
    int* status;
    long long q_stride, num_pages, scratch_floats;
    int max_pages, n_layers, layer, nh, nkv, d, page_size, window, act, form;
    int n_items, n_tiles, total, max_rows, max_keys;
    float scale;
};
static_assert(sizeof(RowCall) == 13 * 8 + 3 * 8 + 15 * 4 + 4, "the caller lays this out field by field");

static int ar_check(const RowCall& c) {
    if (c.nh <= 0 || c.nkv <= 0 || c.nh % c.nkv || c.d <= 0 || c.page_size <= 0 || c.layer < 0 || c.layer >= c.n_layers || c.max_pages <= 0 ||
        c.num_pages <= 0 || !c.status || !(c.scale > 0.f) || c.window < 0 || !aligned16(c.pool) || !aligned16(c.scales))
        return ST_ERR_BAD_ARG;
    if (!ar_types(c.act, c.form)) return ST_ERR_BAD_DTYPE;
    if ((c.form < C8_BF16) != (c.scales != nullptr)) return ST_ERR_BAD_ARG;
    if (c.d > 256 || c.nh > 65535 || c.num_pages > 0x7fffffffll || !c8_rows_fit(c.num_pages, c.n_layers, c.nkv, c.page_size)) return ST_ERR_TOO_LARGE;
    return 0;
}
static PagedKV ar_kv(const RowCall& c) {
    return PagedKV{(const unsigned char*)c.pool, c.scales, c.table, c.max_pages, (int)c.num_pages, c.n_layers, c.layer, c.nkv, c.page_size,
                   c8_shift(c.page_size), c8_reach(c.max_pages, c.page_size), c.status};
}
static SingleArgs ar_single_args(const RowCall& c) {
    SingleArgs a{};
    a.q = c.q; a.out = c.out; a.kv = ar_kv(c); a.items = c.items; a.positions = c.positions; a.seq_of_token = c.seq_of_token;
    a.slots = c.slots; a.nh = c.nh; a.group = c.nh / c.nkv; a.d = c.d; a.n_items = c.n_items; a.scale_log2 = c.scale * AR_LOG2E;
    a.window = c.window;
    return a;
}
static RowArgs ar_row_args(const RowCall& c) {
    RowArgs a{};
    a.q = c.q; a.out = c.out; a.q_stride = c.q_stride > 0 ? c.q_stride : (long long)c.nh * c.d; a.kv = ar_kv(c);
    a.positions = c.positions; a.seq_of_token = c.seq_of_token; a.slots = c.slots; a.d = c.d;
    a.scale_log2 = c.scale * AR_LOG2E; a.window = c.window;
    a.plan = RowPlan{c.tiles, c.items, c.n_tiles, c.total, 0, 0, c.nh, c.nkv, c.nh / c.nkv};
    ar_deal(a, c.act, c.form);
    return a;
}

ST_EXPORT int st_attention_rows_per_tile() { return AR_ROWS; }
ST_EXPORT int st_attention_rows_chunk() { return AR_CHUNK; }
ST_EXPORT int st_attention_rows_unit() { return AR_UNIT; }
// floats of scratch for the parts of a plan's line of `total` places; shared: of its n_tiles x nkv units each
ST_EXPORT long long st_attention_rows_scratch(int n_tiles, int nkv, int d, int total, int shared) {
    if (total <= 0 || d <= 0) return 0;
    const long long walkers = total < ar_walkers_most(d) ? total : ar_walkers_most(d);
    return (shared ? (long long)n_tiles * nkv + walkers : 2 * walkers) * (long long)ar_part_floats(d);
}
// the keys that a single token reads itself, as lo | hi << 32
ST_EXPORT long long st_attention_single8_span(int pos, int window, int shared, int reach) {
    const SingleSpan k = sg_span(pos, window, shared, reach);
    return k.lo | (long long)k.hi << 32;
}
// floats of scratch that single tokens want for this call (0: none), laid out at `from`
static long long ar_line(const RowCall& c, SingleArgs* a, float* from) {
    if (c.nkv <= 0 || c.d <= 0 || !ar_single_fast(c.page_size, c.d, c.form)) return 0;
    const LineShape s = sg_line_shape(c.n_items, c.nh / c.nkv, c.nkv, c.d, c.max_keys, (long long)c.max_pages * c.page_size, c.act == 0, c.form);
    if (!s.walkers) return 0;
    const long long rows = s.slots * s.R, units = s.slots - s.walkers;
    if (a) {
        a->walkers = s.walkers;
        a->line = RowParts{from, from + rows, from + 2 * rows};
        a->span = reinterpret_cast<int*>(from + rows * (2 + c.d));
    }
    return rows * (2 + c.d) + 2 * units;
}
ST_EXPORT long long st_attention_single8_scratch(int n_items, int nh, int nkv, int d, int page_size, int max_pages, int max_keys, int act, int form) {
    RowCall c{};
    c.n_items = n_items; c.nh = nh; c.nkv = nkv; c.d = d; c.page_size = page_size; c.max_pages = max_pages; c.max_keys = max_keys; c.act = act; c.form = form;
    return ar_line(c, nullptr, nullptr);
}

// single tokens; max_keys: about the longest of them (it decides how the work is spread, nothing else)
ST_EXPORT int st_attention_single8(const RowCall* c, void* stream) {
    const int bad = ar_check(*c);
    if (bad) return bad;
    if (c->n_items <= 0) return 0;
    SingleArgs a = ar_single_args(*c);
    if (c->scratch && c->scratch_floats >= ar_line(*c, nullptr, nullptr) && aligned16(c->out) && aligned16(c->scratch)) ar_line(*c, &a, c->scratch);
    return ar_single(a, c->act, c->form, c->max_keys, (cudaStream_t)stream);
}

// tiles of tokens that follow one another in a request
ST_EXPORT int st_attention_tiles8(const RowCall* c, void* stream) {
    const int bad = ar_check(*c);
    if (bad) return bad;
    if (c->n_tiles <= 0 || c->total <= 0) return 0;
    if (c->nh / c->nkv > AR_ROWS) return ST_ERR_TOO_LARGE;
    RowArgs a = ar_row_args(*c);
    const long long slots = 2ll * a.plan.ctas;
    if (c->scratch_floats < slots * (long long)ar_part_floats(c->d)) return ST_ERR_BAD_ARG;
    a.parts = ar_parts(c->scratch, slots);
    a.direct = 1;
    const cudaStream_t s = (cudaStream_t)stream;
    const int r = ar_rows(a, c->act, c->form, c->max_rows, s);
    if (r || a.plan.ctas == 1) return r;
    const dim3 grid(a.plan.ctas, 8);
    return c->act == 0 ? st_launch_pdl("rows_join", attention_rows_join_kernel<float>, grid, dim3(256), 0, s, a)
                       : st_launch_pdl("rows_join", attention_rows_join_kernel<bf16>, grid, dim3(256), 0, s, a);
}

// single tokens in groups that share their first keys: the prefixes' parts, then every token's own keys and the whole
ST_EXPORT int st_attention_shared(const RowCall* c, void* stream) {
    const int bad = ar_check(*c);
    if (bad) return bad;
    if (c->n_items <= 0) return 0;
    if (c->nh / c->nkv > AR_ROWS || c->q_stride > 0) return ST_ERR_BAD_ARG;
    const cudaStream_t s = (cudaStream_t)stream;
    SingleArgs single = ar_single_args(*c);
    long long used = 0;                     // floats of scratch
    if (c->total > 0) {
        RowArgs a = ar_row_args(*c);
        const long long slots = (long long)c->n_tiles * c->nkv + a.plan.ctas;
        if (c->scratch_floats < slots * (long long)ar_part_floats(c->d)) return ST_ERR_BAD_ARG;
        if (slots > (1 << 30) / AR_ROWS) return ST_ERR_TOO_LARGE;
        a.parts = ar_parts(c->scratch, slots);
        a.direct = 0;
        const int r = ar_rows(a, c->act, c->form, c->max_rows, s);
        if (r) return r;
        single.info = c->info;
        single.plan = a.plan;
        single.parts = a.parts;
        used = slots * (long long)ar_part_floats(c->d);
    }
    if (c->scratch && c->scratch_floats >= used + ar_line(*c, nullptr, nullptr) && aligned16(c->out) && aligned16(c->scratch))
        ar_line(*c, &single, c->scratch + used);
    return ar_single(single, c->act, c->form, c->max_keys, s);
}
