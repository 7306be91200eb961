// Attention of tiles of query rows (attention_rows.cuh) over 8-bit and bfloat16 paged caches on tcgen05: portions of prompts, and
// groups of tokens over the prefix they share.
//
// Mathematics: as in attention_single8.cuh.  Codes of an 8-bit cache and queries (scaled by a power of two per row) are halves, the rows'
// scales stay outside: s_j = (q . c_j) ks_j, P_j = p_j vs_j in one half (2^-12 of itself at most, beside results of 2^-9: errors of 0.00167 of
// the norm, of which 0.00165 are the results' rounding); over bfloat16 caches queries, keys and values are bfloat16 and P is two bfloat16
// numbers, both multiplied (one: 0.0018 to 0.0020 of the norm; 16 members behind 2000 keys took 24.0 us then, 25.0 now, 64 behind 8000,
// 32 heads of 64, 50.2 and 54.7).  S = Q K^T of 128 rows x 64 keys and O += P V are tcgen05 products with their sums in tensor memory; P goes there
// straight from the softmax threads' registers (the product's A operand).
//
// One block per SM, in it two groups that have nothing to do with one another: each walks its own run of the plan's chunks in tiles of
// 64 keys, with four softmax warps (a thread per row), a warp that issues its products, two that bring keys and two that bring values
// through two buffers each.  What one group waits for the other fills: a tile is a chain (codes landed, S, softmax, P V) whose
// links are a few hundred to a thousand clocks each.  The next piece's queries are brought by the softmax warps while the last P V
// of a piece is on the tensor cores; its first S then runs under their stores.
//   8-bit forms: neighbouring lanes read a row in 16-byte loads, a tile ahead of the conversion to halves, which is stored in the 128-byte
//   swizzled layout that the matrix descriptors expect.  At head size 128 the two halves of every 16 codes go to different blocks of
//   64 dimensions (rt_place): neighbouring lanes then store to different banks without sorting; queries are stored alike, results
//   are put in order when they leave.
//   bfloat16: asynchronous copies into that layout.
// Page sizes are arbitrary: a lane looks up its row's page two tiles ahead of its loads.
// The warps that bring keys also leave both scales of the rows, the largest value scale of a tile, from which the softmax threads take the
// power of two that keeps P in a half's range (attention_single8.cuh), and a bit per key that has a page.
//
// Bound by the chain of a tile: about 3500 clocks (head size 64) for each of the two groups, where the exponentials of both take 1024 and
// the products 512.  Leaving out exponentials, scales or conversions one at a time changed nothing, all of them together a tenth: the waits and
// hand-overs remain.  2000 tokens of three prompts, 32 heads of 64, int8: 62.5 us with the join; 1000 tokens behind 1500 keys, 32 heads
// of 128, e4m3: 95 us.  The bfloat16 prompt kernel takes 36 and 58 us for the like (attention_prefill_tmap.cu: 2450 clocks a tile).
//
// Waits are bounded; one that expires marks the block dead, the other waits end, `status` gets 3, tensor memory is freed and the
// kernel returns.
#include "attention_rows.cuh"
#include "tcgen05.cuh"

#define RT_THREADS 640                   // 8 softmax warps, 8 bringing keys and values, 2 issuing products, 2 that fill the last four
// Registers a thread keeps after the block has shared them out anew; the sum must not pass what the launch got, 640 x 96.
#define RT_REGS_SOFTMAX 144
#define RT_REGS_BRING 80
#define RT_REGS_ISSUE 32
#define RT_REGS_ALL (256 * RT_REGS_SOFTMAX + 256 * RT_REGS_BRING + 128 * RT_REGS_ISSUE)
static_assert(RT_REGS_ALL <= RT_THREADS * 96, "more registers than the block owns");
#define RT_STAGE 2048                    // bytes a softmax warp's results go through on their way out: 32 rows of 16
#define RT_META 4                        // tiles whose scales are kept: see below

__device__ __forceinline__ void rt_mbar_arrive(uint32_t mbar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(mbar) : "memory");
}
// Named barriers 1-4: a softmax group and the warp that issues its products (160 threads): 0 "S has been read", 1 "P has been
// written".  5: the whole block.  A softmax warp without rows of its own, or one that has given up waiting, meets the issuing warp there
// instead of only arriving, so that it cannot come round twice.
__device__ __forceinline__ void rt_arrive(int wg, int which) {
    const int id = 2 * wg + which;
    if (id == 0) asm volatile("bar.arrive 1, 160;\n" ::: "memory");
    else if (id == 1) asm volatile("bar.arrive 2, 160;\n" ::: "memory");
    else if (id == 2) asm volatile("bar.arrive 3, 160;\n" ::: "memory");
    else asm volatile("bar.arrive 4, 160;\n" ::: "memory");
}
__device__ __forceinline__ void rt_sync(int wg, int which) {
    const int id = 2 * wg + which;
    if (id == 0) asm volatile("bar.sync 1, 160;\n" ::: "memory");
    else if (id == 1) asm volatile("bar.sync 2, 160;\n" ::: "memory");
    else if (id == 2) asm volatile("bar.sync 3, 160;\n" ::: "memory");
    else asm volatile("bar.sync 4, 160;\n" ::: "memory");
}
__device__ __forceinline__ void rt_mul2(float& d0, float& d1, float b0, float b1) {       // d *= b
    asm("{\n\t.reg .b64 b, d;\n\tmov.b64 b, {%2, %3};\n\tmov.b64 d, {%0, %1};\n\tmul.rn.f32x2 d, d, b;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
        : "+f"(d0), "+f"(d1) : "f"(b0), "f"(b1));
}
// bits lo .. hi - 1 of a word
__device__ __forceinline__ uint32_t rt_bits(int lo, int hi) {
    const uint32_t below = hi <= 0 ? 0u : hi >= 32 ? 0xffffffffu : (1u << hi) - 1;
    return lo <= 0 ? below : lo >= 32 ? 0u : below & (0xffffffffu << lo);
}

// the keys of a piece: tiles of 64 from k0 on, below k_end
struct RtKeys { int k0, k_end, n; };
__device__ __forceinline__ RtKeys rt_keys(const RowPiece& p) {
    RtKeys k;
    k.k0 = (p.t.key_lo & ~(AR_CHUNK - 1)) + p.chunk0 * AR_CHUNK;
    k.k_end = min(k.k0 + p.chunks * AR_CHUNK, p.t.key_hi);
    k.n = (k.k_end - k.k0 + TC_BN - 1) / TC_BN;
    return k;
}
// where dimension 8 c + i of a row is kept: piece rt_place(c) + i, in blocks of 64
template <bool HALF, int DP> __device__ __forceinline__ int rt_place(int c) { return HALF && DP == 128 ? (c & 1) * 8 + (c >> 1) : c; }

// what the softmax threads need to know of a tile, beside S
struct RtMeta {
    float ks[RT_META][TC_BN], vs[RT_META][TC_BN];
    float vmax[RT_META][2];              // the largest value scale of each half of the keys
    uint32_t seen[RT_META][2];           // bit c: key c of that half is one of the tile's and has a page
};

// SHARED: tiles of single tokens over the keys that their requests share; else of neighbouring tokens of one request.
template <int FORM, int DP, bool SHARED>
__global__ void __launch_bounds__(RT_THREADS, 1) attention_rows_tc_kernel(const RowArgs a) {
    constexpr bool HALF = FORM != C8_BF16;
    constexpr int DB = DP / 64;                                        // blocks of 64 dimensions
    constexpr uint32_t Q_BLK = TC_BM * 128, KV_BLK = TC_BN * 128;      // bytes of a [rows][64] block
    constexpr uint32_t Q_BUF = DB * Q_BLK, BUF = DB * KV_BLK;
    constexpr uint32_t ALL_BYTES = 2 * Q_BUF + 8 * BUF + 8 * RT_STAGE;
    constexpr int WG_COLS = 256, T_O = 64, T_P = 64 + DP;              // a group's columns: S, O, P (of bfloat16: its first numbers, its second)
    constexpr uint32_t NONE = 0xffffffffu;
    extern __shared__ unsigned char rt_raw[];
    __shared__ __align__(16) RtMeta s_meta[2];
    // per group: S done, O done, "landed" for K0 K1 V0 V1, "free" for the same, queries landed, the scales of four tiles
    __shared__ __align__(8) unsigned long long s_mbar[2][11 + RT_META];
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    __shared__ RowWalk s_walk[2];
    const uint32_t base = (tc_smem(rt_raw) + 1023u) & ~1023u;
    const int tid = threadIdx.x, warp = tc_warp(), lane = tid & 31;
    const int d = a.d, g = a.plan.group;
    {
        uint32_t dyn;
        asm volatile("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn));
        if (base + ALL_BYTES > tc_smem(rt_raw) + dyn) {
            if (tid == 0) atomicExch(a.kv.status, 4);
            return;
        }
    }
    // the group: softmax warps 0-3 and 4-7, the others in turn
    const int wg = warp < 8 ? warp >> 2 : warp & 1;
    const uint32_t sQ = base + wg * Q_BUF;
    auto buf_of = [&](int which) { return base + 2 * Q_BUF + (uint32_t)(wg * 2 + which) * 2 * BUF; };
    auto bar = [&](int i) { return tc_smem(&s_mbar[wg][i]); };
    constexpr int M_S = 0, M_O = 1, M_FULL = 2, M_FREE = 6, M_Q = 10, M_META = 11;
    if (tid == 0) {
        for (int w = 0; w < 2; ++w)
            for (int k = 0; k < 11 + RT_META; ++k)
                tc_mbar_init(tc_smem(&s_mbar[w][k]), k >= M_META || (k >= M_FULL && k < M_FREE) ? 2 : k == M_Q ? 4 : 1);
        tc_mbar_init_fence();
        s_dead = 0;
    }
    if (warp == 1 || warp == 2) {
        RowWalk w;
        w.begin(a.plan, 2 * blockIdx.x + warp - 1);
        if (lane == 0) s_walk[warp - 1] = w;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc_smem(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    ST_PDL_TRIGGER();
    const uint32_t tmem = s_tmem;
    volatile int* dead = &s_dead;
    RowWalk walk = s_walk[wg];
    RowPiece pc;

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(RT_REGS_ISSUE));
        if (warp < 18) {
            // ---- the warp that issues the group's products
            const uint32_t t_wg = tmem + wg * WG_COLS;
            constexpr uint32_t type = HALF ? 0u : (1u << 7) | (1u << 10);
            constexpr uint32_t idesc_s = (1u << 4) | type | ((TC_BN / 8) << 17) | ((TC_BM / 16) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | type | (1u << 16) | ((DP / 8) << 17) | ((TC_BM / 16) << 24);
            const uint64_t dq = tc_desc(sQ, 16, 1024), dk = tc_desc(buf_of(0), 16, 1024), dv = tc_desc(buf_of(1), KV_BLK, 1024);
            const uint32_t mb_s = bar(M_S), mb_o = bar(M_O), mb_full = bar(M_FULL), mb_free = bar(M_FREE);
            bool alive = true;
            uint32_t n = 0;              // tiles so far: buffer n & 1, phase (n >> 1) & 1
            for (int k = 0; walk.next(a.plan, pc); ++k) {
                const int tiles = rt_keys(pc).n;
                auto issue_s = [&](uint32_t x) {
                    const int b = x & 1;
                    if (alive) alive = tc_wait_warp(mb_full + 8 * b, (x >> 1) & 1, dead);
                    if (alive) {
                        tc_fence_after_sync();
                        if (tc_elect()) {
#pragma unroll
                            for (int kk = 0; kk < DP / 16; ++kk)
                                tc_mma(t_wg, dq + (((kk >> 2) * Q_BLK + (kk & 3) * 32) >> 4),
                                       dk + ((b * BUF + (kk >> 2) * KV_BLK + (kk & 3) * 32) >> 4), idesc_s, kk > 0);
                            tc_commit(mb_s);
                            tc_commit(mb_free + 8 * b);
                        }
                    }
                    __syncwarp();
                };
                if (alive) alive = tc_wait_warp(bar(M_Q), k & 1, dead);
                issue_s(n);
                for (int i = 0; i < tiles; ++i) {
                    const uint32_t x = n + i;
                    const int b = x & 1;
                    rt_sync(wg, 0);      // S(i) is in the softmax threads' registers
                    if (i + 1 < tiles) issue_s(x + 1);
                    rt_sync(wg, 1);      // P(i) is written, O += P V of tile i - 1 has completed
                    if (alive) alive = tc_wait_warp(mb_full + 8 * (2 + b), (x >> 1) & 1, dead);
                    if (alive) {
                        tc_fence_after_sync();
                        if (tc_elect()) {
#pragma unroll
                            for (int jj = 0; jj < TC_BN / 16; ++jj) {
                                tc_mma_ts(t_wg + T_O, t_wg + T_P + jj * 8, dv + ((b * BUF + jj * 2048) >> 4), idesc_o, i > 0 || jj > 0);
                                if (!HALF) tc_mma_ts(t_wg + T_O, t_wg + T_P + TC_BN / 2 + jj * 8, dv + ((b * BUF + jj * 2048) >> 4), idesc_o, 1);
                            }
                            tc_commit(mb_o);
                            tc_commit(mb_free + 8 * (2 + b));
                        }
                    }
                    __syncwarp();
                }
                n += tiles;
            }
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(RT_REGS_BRING));
        // ---- two warps bring the group's keys (which = 0), two its values: 32 rows of every tile each
        const int which = (warp >> 1) & 1, half = (warp - 8) >> 2, row = half * 32 + lane;
        const uint32_t mb_full = bar(M_FULL + which * 2), mb_free = bar(M_FREE + which * 2), mb_meta = bar(M_META);
        const uint32_t buf0 = buf_of(which) + half * 32 * 128;
        RtMeta& meta = s_meta[wg];
        const uint32_t to_values = (uint32_t)a.kv.nkv * a.kv.page_size;
        uint32_t n = 0;                  // tiles so far
        RtKeys keys;
        keys.n = 0;
        RowTable table{nullptr, 1, 0};
        int i = 0;                       // the next tile of the piece
        bool have = true;
        // A lane looks up the page of its row two tiles ahead (ask), turns it into a row of the pool one tile ahead (resolve).
        int page = -1, off = 0, head = 0;
        bool wanted = false;
        auto ask = [&]() {
            wanted = false;
            if (i >= keys.n) {
                if (!walk.next(a.plan, pc)) { have = false; return; }
                keys = rt_keys(pc);
                table = ar_table<SHARED>(a, pc.t);
                head = pc.head;
                i = 0;
            }
            const int key = keys.k0 + TC_BN * i + row;
            ++i;
            const int* const from = ar_row_of<SHARED>(a, pc.t, table, key, key >= pc.t.key_lo && key < keys.k_end);
            if (from) {
                const int index = a.kv.page_index(key);
                wanted = true;
                off = a.kv.offset(key, index);
                page = index < a.kv.max_pages ? __ldg(from + index) : -1;
            }
        };
        uint32_t at = NONE;              // the lane's row among the keys
        bool hole = false;               // a key that a row may see has no page
        auto resolve = [&]() {
            const bool there = (unsigned)page < (unsigned)a.kv.num_pages;
            at = wanted && there ? a.kv.row0(page, 0, head) + off : NONE;
            hole = wanted && !there;
            if (!SHARED && hole) hole = ar_needed(a, pc.t, keys.k0 + TC_BN * (i - 1) + row);
        };
        // Scales and marks of a tile, into the place of its turn.  RT_META places: the tile four before has been read when this one's key
        // buffer is free, because S of the tile two before was issued after the softmax threads were done with the one before that.
        auto put_meta = [&](float ks, float vs) {
            const int x = n & (RT_META - 1);
            if (HALF) {
                // (a value row that is not finite has the scale NaN: with the key's it reaches those who see the key and nobody else)
                meta.ks[x][row] = isnan(vs) ? vs : ks;
                vs = isnan(vs) ? 0.f : vs;
                meta.vs[x][row] = vs;
                const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(vs));
                if (lane == 0) meta.vmax[x][half] = __uint_as_float(most);
            }
            const uint32_t seen = __ballot_sync(0xffffffffu, at != NONE);
            __syncwarp();
            if (lane == 0) {
                meta.seen[x][half] = seen;
                rt_mbar_arrive(mb_meta + 8 * x);
            }
            if (hole) *a.kv.status = 1;
        };
        auto landed = [&](uint32_t x) {
            tc_fence_async_smem();
            __syncwarp();
            if (lane == 0) rt_mbar_arrive(mb_full + 8 * (x & 1));
        };
        auto wait_free = [&]() -> bool { return n < 2 || tc_wait_warp(mb_free + 8 * (n & 1), ((n - 2) >> 1) & 1, dead); };
        ask();
        const unsigned char* pool = a.kv.pool + (which ? (size_t)to_values * d * c8_bytes(FORM) : 0);
        if constexpr (HALF) {
            // NP neighbouring lanes read a row, 16 bytes each: load j has rows j RI .. j RI + RI - 1 of the warp's 32
            constexpr int NP = DP / 16, RI = 32 / NP;
            const int p = lane % NP, rl = lane / NP;
            const bool in = 16 * p < d;
            const unsigned char* mine = pool + 16 * p;
            // the 16-byte pieces (eight halves) of a row's codes 16 p .. 16 p + 15, for even and odd j (at RI = 4 the rows' swizzle differs)
            const int c0 = rt_place<true, DP>(2 * p), c1 = rt_place<true, DP>(2 * p + 1);
            const uint32_t to0 = buf0 + rl * 128 + (c0 >> 3) * KV_BLK, to1 = buf0 + rl * 128 + (c1 >> 3) * KV_BLK;
            const uint32_t even0 = to0 + (((c0 & 7) ^ (rl & 7)) << 4), even1 = to1 + (((c1 & 7) ^ (rl & 7)) << 4);
            const uint32_t odd0 = to0 + (((c0 & 7) ^ ((rl + RI) & 7)) << 4), odd1 = to1 + (((c1 & 7) ^ ((rl + RI) & 7)) << 4);
            uint4 data[NP];
            float ks = 0.f, vs = 0.f;
            auto load = [&]() {
                uint32_t r[NP];
#pragma unroll
                for (int j = 0; j < NP; ++j) r[j] = __shfl_sync(0xffffffffu, at, j * RI + rl);
#pragma unroll
                for (int j = 0; j < NP; ++j)
                    data[j] = in && r[j] != NONE ? __ldg(reinterpret_cast<const uint4*>(mine + (size_t)r[j] * d)) : make_uint4(0u, 0u, 0u, 0u);
                if (which == 0) {
                    ks = at != NONE ? __ldg(a.kv.scales + at) : 0.f;
                    vs = at != NONE ? __ldg(a.kv.scales + at + to_values) : 0.f;
                }
            };
            bool now = have;                                 // there is a tile in the registers
            if (now) {
                resolve();
                load();
                ask();
            }
            while (now) {
                if (!wait_free()) break;
                if (which == 0) put_meta(ks, vs);
                const uint32_t b = (n & 1) * BUF;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    uint32_t h[8];
                    c8_halves<FORM>(data[j].x, h[0], h[1]);
                    c8_halves<FORM>(data[j].y, h[2], h[3]);
                    c8_halves<FORM>(data[j].z, h[4], h[5]);
                    c8_halves<FORM>(data[j].w, h[6], h[7]);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n"
                                 ::"r"((j & 1 ? odd0 : even0) + b + j * RI * 128), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n"
                                 ::"r"((j & 1 ? odd1 : even1) + b + j * RI * 128), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
                }
                now = have;
                if (now) {
                    resolve();
                    load();                                  // under way while this tile is announced and its successor's buffer waited for
                    ask();
                }
                landed(n);
                ++n;
            }
        } else {
            // copies of a tile are asked for as soon as its buffer is free; the tile before is announced when its own have landed
            constexpr int NP = DP / 8, RI = 32 / NP;         // lanes of a row, rows of a copy
            const int p = lane % NP, rl = lane / NP;
            const bool in = 8 * p < d;
            bool alive = true;
            while (have) {
                resolve();
                ask();
                if (!wait_free()) { alive = false; break; }
                if (which == 0) put_meta(0.f, 0.f);
                const uint32_t buf = buf0 + (n & 1) * BUF + (p >> 3) * KV_BLK;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const int row_j = j * RI + rl;
                    const uint32_t r = __shfl_sync(0xffffffffu, at, row_j);
                    const bool ok = in && r != NONE;
                    tc_cp16(buf + row_j * 128 + (((p & 7) ^ (row_j & 7)) << 4), ok ? pool + (size_t)r * d * 2 + 16 * p : pool, ok);
                }
                tc_cp_commit();
                ++n;
                if (n > 1) {
                    tc_cp_wait<1>();
                    landed(n - 2);
                }
            }
            tc_cp_wait<0>();
            if (alive && n > 0) landed(n - 1);
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(RT_REGS_SOFTMAX));
        // ---- softmax threads: thread `row` of a group has query row `row`, a lane of tensor memory
        const int row = tid & 127, warp4 = warp & 3;
        const uint32_t t_wg = tmem + wg * WG_COLS + ((uint32_t)(warp4 * 32) << 16);
        const uint32_t mb_s = bar(M_S), mb_o = bar(M_O), mb_meta = bar(M_META);
        const RtMeta& meta = s_meta[wg];
        bool alive = true;
        uint32_t n = 0;                                  // tiles so far
        // ---- queries.  A piece's tokens and positions are looked up a piece ahead.
        RowPiece nx;
        int token_n = -1, pos_n = -1;
        auto look = [&]() -> bool {
            if (!walk.next(a.plan, nx)) return false;
            const int place = nx.t.first + row / g;
            token_n = row < nx.t.n_tok * g ? (SHARED ? __ldg(a.plan.items + place) : place) : -1;
            pos_n = token_n >= 0 ? __ldg(a.positions + token_n) : -1;
            if (token_n >= 0) {                          // the row's lines, for `bring`
                const bf16* q = (const bf16*)a.q + (size_t)token_n * a.q_stride + (nx.head * g + row % g) * d;
                asm volatile("prefetch.global.L1 [%0];\n" ::"l"(q));
                if (DP == 128) asm volatile("prefetch.global.L1 [%0];\n" ::"l"(q + (d > 64 ? 64 : 0)));
            }
            return true;
        };
        // The warp's 32 rows of `nx` into shared memory: NP neighbouring lanes have a row, RI rows to a load.  All S over the queries
        // that were there are complete.  Returns the factor of this thread's row.
        auto bring = [&]() -> float {
            constexpr int NP = DP / 8, RI = 32 / NP;
            float fac = a.scale_log2;
            if (warp4 * 32 < nx.t.n_tok * g) {
                const int p = lane % NP, rl = lane / NP;
                const int r_own = pos_n >= 0 ? row % g : 0;
                const long long at_own = pos_n >= 0 ? (long long)token_n * a.q_stride + (nx.head * g + r_own) * d : -1;
                uint4 u[NP];
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const long long at = __shfl_sync(0xffffffffu, at_own, j * RI + rl);
                    u[j] = at >= 0 && 8 * p < d ? __ldg(reinterpret_cast<const uint4*>((const bf16*)a.q + at) + p) : make_uint4(0u, 0u, 0u, 0u);
                }
                const int place = rt_place<HALF, DP>(p);
                const uint32_t dst = sQ + (place >> 3) * Q_BLK;
                int ex_own = 0;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const int r = warp4 * 32 + j * RI + rl;
                    uint32_t* w = &u[j].x;
                    if (HALF) {
                        // a power of two that brings the row's largest element to [2^14, 2^15)
                        uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
#pragma unroll
                        for (int o = NP / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
                        const int ex = min(max((int)(max(m & 0xffffu, m >> 16) >> 7) - 127, -100), 127);
                        const int theirs = __shfl_sync(0xffffffffu, ex, (lane % RI) * NP);
                        if (lane / RI == j) ex_own = theirs;
                        const float mul = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const __half2 h = __floats2half2_rn(__uint_as_float(w[i] << 16) * mul, __uint_as_float(w[i] & 0xffff0000u) * mul);
                            w[i] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                    }
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n"
                                 ::"r"(dst + r * 128 + (((place & 7) ^ (r & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                }
                if (HALF) fac = ldexpf(a.scale_log2, ex_own - 14);
                tc_fence_async_smem();
                __syncwarp();
            }
            if (lane == 0) rt_mbar_arrive(bar(M_Q));
            return fac;
        };
        bool more = look();
        float fac_n = more ? bring() : 0.f;
        while (more) {
            pc = nx;
            const RtKeys keys = rt_keys(pc);
            const int rows = pc.t.n_tok * g, pos = pos_n, token = token_n;
            const float fac = fac_n;
            more = look();
            if (warp4 * 32 >= rows) {                    // no row of this warp's is one of the tile's
                for (int i = 0; i < keys.n; ++i) { rt_sync(wg, 0); rt_sync(wg, 1); }
                n += keys.n;
                if (more) fac_n = bring();
                continue;
            }
            const int hi = min(pos, keys.k_end - 1) + 1;
            const int lo = max(pc.t.key_lo, a.window > 0 ? pos - a.window + 1 : 0);
            float ref = -INFINITY, sum = 0.f;
            for (int i = 0; i < keys.n; ++i) {
                const uint32_t x = n + i;
                const int key0 = keys.k0 + TC_BN * i, mt = x & (RT_META - 1);
                if (alive) alive = tc_wait_warp(mb_s, x & 1, dead);
                tc_fence_after_sync();
                float s[TC_BN];
                tc_ld32(t_wg, s);
                tc_ld32(t_wg + 32, s + 32);
                if (alive) alive = tc_wait_warp(mb_meta + 8 * mt, (x / RT_META) & 1, dead);
                tc_ld_wait();
                tc_fence_before_sync();
                if (alive) rt_arrive(wg, 0);
                else rt_sync(wg, 0);
                if (HALF) {
#pragma unroll
                    for (int c = 0; c < TC_BN; c += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&meta.ks[mt][c]);
                        rt_mul2(s[c], s[c + 1], f.x, f.y);
                        rt_mul2(s[c + 2], s[c + 3], f.z, f.w);
                    }
                }
                float vmax = HALF ? fmaxf(meta.vmax[mt][0], meta.vmax[mt][1]) : 0.f;
                const uint2 seen = *reinterpret_cast<const uint2*>(meta.seen[mt]);
                if ((seen.x & seen.y) != 0xffffffffu || key0 + TC_BN > hi || key0 < lo) {
                    // this row does not see all 64 keys
                    const uint32_t b0 = seen.x & rt_bits(lo - key0, hi - key0), b1 = seen.y & rt_bits(lo - key0 - 32, hi - key0 - 32);
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        if (!(b0 >> c & 1)) s[c] = -INFINITY;
                        if (!(b1 >> c & 1)) s[c + 32] = -INFINITY;
                    }
                    if (HALF) {
                        // the scale of a key that the row does not see has no part in its unit
                        vmax = 0.f;
#pragma unroll
                        for (int c = 0; c < TC_BN; c += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(&meta.vs[mt][c]);
                            const uint32_t b = (c < 32 ? b0 : b1) >> (c & 31);
                            vmax = tc_max3(vmax, b & 1 ? f.x : 0.f, b & 2 ? f.y : 0.f);
                            vmax = tc_max3(vmax, b & 4 ? f.z : 0.f, b & 8 ? f.w : 0.f);
                        }
                    }
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < TC_BN; c += 8) {
                    mx4[0] = tc_max3(mx4[0], s[c], s[c + 1]); mx4[1] = tc_max3(mx4[1], s[c + 2], s[c + 3]);
                    mx4[2] = tc_max3(mx4[2], s[c + 4], s[c + 5]); mx4[3] = tc_max3(mx4[3], s[c + 6], s[c + 7]);
                }
                const float lead = HALF ? (float)max((int)(__float_as_uint(vmax) >> 23) - 126, -90) : 0.f;
                const float need = fmaf(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), fac, lead);
                // the reference moves when p vs could pass 2^15 (or from "no key yet"), and then to 11 below the largest
                const bool move = need > ref + 15.f;
                const float old = ref;
                if (move) ref = need - 11.f;
                const float neg = ref == -INFINITY ? 0.f : -ref;
                float rs[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                uint32_t w[TC_BN / 2], w2[HALF ? 1 : TC_BN / 2];
#pragma unroll
                for (int c = 0; c < TC_BN; c += 4) {
                    float p[4];
                    tc_fma2(p[0], p[1], s[c], s[c + 1], fac, neg);
                    tc_fma2(p[2], p[3], s[c + 2], s[c + 3], fac, neg);
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = tc_exp2(p[j]);
                    tc_add2(rs[c & 4], rs[(c & 4) + 1], p[0], p[1]);
                    tc_add2(rs[(c & 4) + 2], rs[(c & 4) + 3], p[2], p[3]);
                    if (HALF) {
                        const float4 f = *reinterpret_cast<const float4*>(&meta.vs[mt][c]);
                        rt_mul2(p[0], p[1], f.x, f.y);
                        rt_mul2(p[2], p[3], f.z, f.w);
                        const __half2 h0 = __floats2half2_rn(p[0], p[1]), h1 = __floats2half2_rn(p[2], p[3]);
                        w[c / 2] = *reinterpret_cast<const uint32_t*>(&h0);
                        w[c / 2 + 1] = *reinterpret_cast<const uint32_t*>(&h1);
                    } else {
                        // p in two numbers: one of 2^-8 would be the largest error of the result
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const __nv_bfloat162 first = __floats2bfloat162_rn(p[2 * h], p[2 * h + 1]);
                            const uint32_t u = *reinterpret_cast<const uint32_t*>(&first);
                            const __nv_bfloat162 rest = __floats2bfloat162_rn(p[2 * h] - __uint_as_float(u << 16), p[2 * h + 1] - __uint_as_float(u & 0xffff0000u));
                            w[c / 2 + h] = u;
                            w2[c / 2 + h] = *reinterpret_cast<const uint32_t*>(&rest);
                        }
                    }
                }
                if (i > 0) {                             // O += P V of tile i - 1: O may be scaled and P overwritten after it
                    if (alive) alive = tc_wait_warp(mb_o, (x - 1) & 1, dead);
                    tc_fence_after_sync();
                }
                if (__any_sync(0xffffffffu, move) && i > 0) {
                    const float corr = move ? tc_exp2(old - ref) : 1.f;
#pragma unroll
                    for (int cb = 0; cb < DP / 32; ++cb) {
                        float ov[32];
                        tc_ld32(t_wg + T_O + cb * 32, ov);
                        tc_ld_wait();
#pragma unroll
                        for (int kk = 0; kk < 32; ++kk) ov[kk] *= corr;
                        tc_st32(t_wg + T_O + cb * 32, ov);
                    }
                    tc_st_wait();
                    sum *= corr;
                }
                tc_st32(t_wg + T_P, reinterpret_cast<const float*>(w));
                if constexpr (!HALF) tc_st32(t_wg + T_P + TC_BN / 2, reinterpret_cast<const float*>(w2));
                sum += ((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7]));
                tc_st_wait();
                tc_fence_before_sync();
                if (alive) rt_arrive(wg, 1);
                else rt_sync(wg, 1);
            }
            if (more) fac_n = bring();
            if (alive) alive = tc_wait_warp(mb_o, (n + keys.n - 1) & 1, dead);
            tc_fence_after_sync();
            n += keys.n;
            // ---- the piece's sums: out, or into its slot.  Sixteen dimensions at a time change hands in shared memory, so that
            // neighbouring lanes store a row's neighbouring pieces (a thread's own row has a line of its own in every store).
            const bool direct = a.direct && pc.whole;
            const size_t slot0 = (size_t)ar_slot(a, pc, 2 * blockIdx.x + wg) * AR_ROWS;
            if (!direct && row < rows) { a.parts.r[slot0 + row] = ref; a.parts.l[slot0 + row] = sum; }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const bool store = row < rows && pos >= 0 && alive;
            // rows that this lane stores: direct 16 i + lane / 2 (two lanes a row), else 8 i + lane / 4
            const long long mine = store ? direct ? ((long long)token * a.plan.nh + pc.head * g + row % g) * d : (long long)(slot0 + row) * d : -1;
            long long to[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                to[i] = __shfl_sync(0xffffffffu, mine, direct ? (16 * i + (lane >> 1)) & 31 : 8 * i + (lane >> 2));
            const uint32_t stage = base + 2 * Q_BUF + 8 * BUF + warp * RT_STAGE;
#pragma unroll
            for (int cb = 0; cb < DP / 16; ++cb) {
                float o[16];
                __syncwarp();
                tc_ld16(t_wg + T_O + cb * 16, o);
                tc_ld_wait();
                // row `lane`: four pieces of 16 bytes, turned by the row so that eight lanes hit all banks
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};\n"
                                 ::"r"(stage + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)), "f"(direct ? o[4 * c] * inv : o[4 * c]),
                                   "f"(direct ? o[4 * c + 1] * inv : o[4 * c + 1]), "f"(direct ? o[4 * c + 2] * inv : o[4 * c + 2]),
                                   "f"(direct ? o[4 * c + 3] * inv : o[4 * c + 3]) : "memory");
                __syncwarp();
                auto read = [&](int r, int c) -> float4 {
                    float4 v;
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                                 : "r"(stage + r * 64 + ((c ^ ((r >> 1) & 3)) << 4)) : "memory");
                    return v;
                };
                // the eight dimensions that are kept at place 2 cb + c
                auto dim = [&](int c) { const int at = 2 * cb + c; return 8 * (HALF && DP == 128 ? (at & 7) * 2 + (at >> 3) : at); };
                if (direct) {
                    const int c = lane & 1, e = c ? dim(1) : dim(0);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = 16 * i + (lane >> 1);
                        const float4 x = read(r, 2 * c), y = read(r, 2 * c + 1);
                        if (to[i] < 0 || e >= d) continue;
                        const __nv_bfloat162 b[4] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w), __floats2bfloat162_rn(y.x, y.y),
                                                     __floats2bfloat162_rn(y.z, y.w)};
                        *reinterpret_cast<uint4*>((bf16*)a.out + to[i] + e) = *reinterpret_cast<const uint4*>(b);
                    }
                } else {
                    const int c = lane & 3, e = (c >> 1 ? dim(1) : dim(0)) + (c & 1) * 4;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 v = read(8 * i + (lane >> 2), c);
                        if (to[i] >= 0 && e < d) store4(a.parts.o + to[i] + e, v);
                    }
                }
            }
            tc_fence_before_sync();
        }
    }
    tc_fence_before_sync();
    __syncwarp();
    asm volatile("bar.sync 5, %0;\n" ::"n"(RT_THREADS) : "memory");
    if (s_dead && tid == 0) atomicExch(a.kv.status, 3);
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}

template <int FORM, int DP, bool SHARED> static int rt_run(const RowArgs& a, cudaStream_t s) {
    constexpr size_t smem = 2 * (DP / 64) * TC_BM * 128 + 8 * (DP / 64) * TC_BN * 128 + 8 * RT_STAGE + 1024;
    auto kernel = attention_rows_tc_kernel<FORM, DP, SHARED>;
    AR_ALLOW_SMEM(kernel, smem);
    // the redistribution of registers moves what the launch got, and waits for more for ever: only for a kernel compiled as assumed
    static std::atomic<int> regs[64];
    std::atomic<int>& have = regs[ar_device()];
    if (!have) {
        cudaFuncAttributes attr;
        const cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
        if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
        have = attr.numRegs;
    }
    if (have * RT_THREADS < RT_REGS_ALL) return ST_ERR_TOO_LARGE;
    kernel<<<(a.plan.ctas + 1) / 2, RT_THREADS, smem, s>>>(a);
    return st_launch_status();
}

template <int FORM> static int rt_run(const RowArgs& a, cudaStream_t s) {
    if (a.plan.items) return a.d <= 64 ? rt_run<FORM, 64, true>(a, s) : rt_run<FORM, 128, true>(a, s);
    if constexpr (FORM != C8_BF16) return a.d <= 64 ? rt_run<FORM, 64, false>(a, s) : rt_run<FORM, 128, false>(a, s);
    return ST_ERR_BAD_DTYPE;             // portions over bfloat16 caches have kernels of their own
}
int ar_rows_tc(const RowArgs& a, int form, cudaStream_t s) {
    if (form == C8_INT8) return rt_run<C8_INT8>(a, s);
    if (form == C8_E4M3) return rt_run<C8_E4M3>(a, s);
    return rt_run<C8_BF16>(a, s);
}
