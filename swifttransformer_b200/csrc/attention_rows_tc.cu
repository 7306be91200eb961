// Attention of tiles of query rows (attention_rows.cuh) over 8-bit and bfloat16 paged caches on tcgen05: portions of prompts, and
// groups of tokens over the prefix they share.
//
// Mathematics: as in attention_single8.cuh.  Codes of an 8-bit cache and queries (scaled by a power of two per row) are halves, the rows'
// scales stay outside: s_j = (q . c_j) ks_j, P_j = p_j vs_j in half; over bfloat16 caches queries, keys, P and values are
// bfloat16.  S = Q K^T of 128 rows x 64 keys and O += P V are tcgen05 products with their sums in tensor memory; P goes there
// straight from the softmax threads' registers (the product's A operand).
//
// One block per SM walks its run of the plan's chunks.  Two groups of four softmax warps take every second tile of 64 keys of a
// piece, each with its own S, O and P in tensor memory, key and value buffers (two each) and issuing warp; at the piece's end
// the first group reads the second's O from tensor memory (the lanes are the same rows) and stores the sum.  Four warps bring
// keys, four bring values, for both groups in turn, and run ahead across pieces:
//   8-bit forms: 16-byte loads to registers, several tiles ahead (32 KB per SM under way: memory needs that), conversion to
//   halves, stores into the 128-byte swizzled layout the matrix descriptors expect.  Conversion is the price of the format: about
//   2.5 instructions per four codes against the softmax's 4 per score; with one row of 128 codes per thread, two warps each, it
//   bounded the kernel, so there are four.
//   bfloat16: asynchronous copies into that layout, as many tiles ahead as there are buffers.
// Page sizes are arbitrary: every thread looks up its row's page, a tile ahead of its loads.
// With the row's scales go their largest value scale per tile, from which the softmax threads take the power of two that keeps P in
// a half's range (attention_single8.cuh), and a mark where a key has no page.
//
// Bound by the softmax (an exponential per score, 16 a clock and SM) at head size 64, by softmax and conversion together at 128, and by
// memory for prefixes shared by few rows.  Waits are bounded; one that expires marks the block dead, the other waits end, `status`
// gets 3, tensor memory is freed and the kernel returns.
#include "attention_rows.cuh"
#include "tcgen05.cuh"

#define RT_THREADS 640                   // 8 softmax warps, 4 for keys, 4 for values, 2 issuing products, 2 for queries
// Registers a thread keeps after the block has shared them out anew; the sum must not pass what the launch got, 640 x 96.
#define RT_REGS_SOFTMAX 144
#define RT_REGS_OTHER 64
static_assert(256 * RT_REGS_SOFTMAX + 384 * RT_REGS_OTHER <= RT_THREADS * 96, "more registers than the block owns");
#define RT_META 4                        // tiles whose scales are kept: see below

__device__ __forceinline__ void rt_mbar_arrive(uint32_t mbar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(mbar) : "memory");
}
// Named barriers.  1-4: a softmax group and the warp that issues its products (160 threads): 0 "S has been read", 1 "P has been written".
// 5: the second group's share of a piece is complete.  6: the first group has read it.  7: the whole block.  A softmax warp that has given up waiting meets the issuing
// warp at 1-4 instead of only arriving, so that it cannot come round twice.
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
__device__ __forceinline__ void rt_share_arrive() { asm volatile("bar.arrive 5, 256;\n" ::: "memory"); }
__device__ __forceinline__ void rt_share_sync() { asm volatile("bar.sync 5, 256;\n" ::: "memory"); }
__device__ __forceinline__ void rt_taken_arrive() { asm volatile("bar.arrive 6, 256;\n" ::: "memory"); }
__device__ __forceinline__ void rt_taken_sync() { asm volatile("bar.sync 6, 256;\n" ::: "memory"); }

__device__ __forceinline__ void rt_mul2(float& d0, float& d1, float b0, float b1) {       // d *= b
    asm("{\n\t.reg .b64 b, d;\n\tmov.b64 b, {%2, %3};\n\tmov.b64 d, {%0, %1};\n\tmul.rn.f32x2 d, d, b;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
        : "+f"(d0), "+f"(d1) : "f"(b0), "f"(b1));
}
// what the softmax threads need to know of a row
struct RtRows {
    int pos[AR_ROWS], token[AR_ROWS];
    float fac[AR_ROWS];
};
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
__device__ __forceinline__ int rt_share(int n, int wg) { return (n - wg + 1) >> 1; }    // tiles of a group

// what the softmax threads need to know of a tile, beside S
struct RtMeta {
    float ks[RT_META][TC_BN], vs[RT_META][TC_BN];
    float vmax[RT_META][2];              // the largest value scale of each half of the keys
    uint32_t seen[RT_META][2];           // bit c: key c of that half is one of the tile's and has a page
};

template <int FORM, int DP>
__global__ void __launch_bounds__(RT_THREADS, 1) attention_rows_tc_kernel(const RowArgs a) {
    constexpr bool HALF = FORM != C8_BF16;
    constexpr int DB = DP / 64;                                        // blocks of 64 dimensions
    constexpr uint32_t Q_BLK = TC_BM * 128, KV_BLK = TC_BN * 128;      // bytes of a [rows][64] block
    constexpr uint32_t Q_BUF = DB * Q_BLK, BUF = DB * KV_BLK;
    constexpr uint32_t ALL_BYTES = 2 * Q_BUF + 8 * BUF;
    constexpr int WG_COLS = 256, T_O = 64, T_P = 64 + DP;              // a group's columns: S, O, P
    extern __shared__ unsigned char rt_raw[];
    __shared__ __align__(16) RtMeta s_meta[2];
    __shared__ RtRows s_rows[2];
    __shared__ float s_mrg[2][128];
    // per group: S done, O done, "landed" for K0 K1 V0 V1, "free" for the same, and the scales of four tiles; of the two
    // query buffers: "landed" and "free"
    __shared__ __align__(8) unsigned long long s_mbar[2][10 + RT_META], s_qbar[2][2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    __shared__ RowWalk s_walk;
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
    const uint32_t sQ = base;                                          // two query buffers
    auto buf_of = [&](int wg, int which, int b) { return base + 2 * Q_BUF + (uint32_t)((wg * 2 + which) * 2 + b) * BUF; };
    auto bar = [&](int wg, int i) { return tc_smem(&s_mbar[wg][i]); };
    constexpr int M_S = 0, M_O = 1, M_FULL = 2, M_FREE = 6, M_META = 10;
    if (tid == 0) {
        for (int w = 0; w < 2; ++w) {
            for (int k = 0; k < 10 + RT_META; ++k)
                tc_mbar_init(bar(w, k), k >= M_META ? (HALF ? 4 : 2) : k >= M_FULL && k < M_FREE ? 2 : 1);
        }
        for (int k = 0; k < 2; ++k) {
            tc_mbar_init(tc_smem(&s_qbar[0][k]), 2);           // both bringing warps
            tc_mbar_init(tc_smem(&s_qbar[1][k]), 2 + 8);       // both groups' last S, all softmax warps
        }
        tc_mbar_init_fence();
        s_dead = 0;
    }
    if (tid == 32) s_walk.begin(a.plan, blockIdx.x);
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
    auto tile_addr = [](uint32_t tile, int r, int c) -> uint32_t { return tile + r * 128 + (((c & 7) ^ (r & 7)) << 4); };

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(RT_REGS_OTHER));
        if (warp < 18) {
            // ---- the warp that issues a group's products
            const int wg = warp - 16;
            const uint32_t t_wg = tmem + wg * WG_COLS;
            constexpr uint32_t type = HALF ? 0u : (1u << 7) | (1u << 10);
            constexpr uint32_t idesc_s = (1u << 4) | type | ((TC_BN / 8) << 17) | ((TC_BM / 16) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | type | (1u << 16) | ((DP / 8) << 17) | ((TC_BM / 16) << 24);
            const uint64_t dk = tc_desc(buf_of(wg, 0, 0), 16, 1024), dv = tc_desc(buf_of(wg, 1, 0), KV_BLK, 1024);
            const uint32_t mb_s = bar(wg, M_S), mb_o = bar(wg, M_O), mb_full = bar(wg, M_FULL), mb_free = bar(wg, M_FREE);
            bool alive = true;
            uint32_t n = 0;              // tiles of this group so far: buffer n & 1, phase (n >> 1) & 1
            RowWalk walk = s_walk;
            RowPiece pc;
            for (int k = 0; walk.next(a.plan, pc); ++k) {
                const int mine = rt_share(rt_keys(pc).n, wg);
                const uint64_t dq = tc_desc(sQ + (k & 1) * Q_BUF, 16, 1024);
                auto issue_s = [&](uint32_t x, bool last) {
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
                            if (last) tc_commit(tc_smem(&s_qbar[1][k & 1]));
                        }
                    }
                    __syncwarp();
                };
                if (alive) alive = tc_wait_warp(tc_smem(&s_qbar[0][k & 1]), (k >> 1) & 1, dead);
                if (mine > 0) issue_s(n, mine == 1);
                else if (lane == 0) rt_mbar_arrive(tc_smem(&s_qbar[1][k & 1]));
                for (int i = 0; i < mine; ++i) {
                    const uint32_t x = n + i;
                    const int b = x & 1;
                    rt_sync(wg, 0);      // S(i) is in the softmax threads' registers
                    if (i + 1 < mine) issue_s(x + 1, i + 2 == mine);
                    rt_sync(wg, 1);      // P(i) is written, O += P V of tile i - 1 has completed
                    if (alive) alive = tc_wait_warp(mb_full + 8 * (2 + b), (x >> 1) & 1, dead);
                    if (alive) {
                        tc_fence_after_sync();
                        if (tc_elect()) {
#pragma unroll
                            for (int jj = 0; jj < TC_BN / 16; ++jj)
                                tc_mma_ts(t_wg + T_O, t_wg + T_P + jj * 8, dv + ((b * BUF + jj * 2048) >> 4), idesc_o, i > 0 || jj > 0);
                            tc_commit(mb_o);
                            tc_commit(mb_free + 8 * (2 + b));
                        }
                    }
                    __syncwarp();
                }
                n += mine;
            }
        } else {
            // ---- two warps bring the queries, a piece ahead: a thread has two rows
            RowWalk walk = s_walk;
            RowPiece pc;
            for (int k = 0; walk.next(a.plan, pc); ++k) {
                if (k >= 2 && !tc_wait_warp(tc_smem(&s_qbar[1][k & 1]), ((k - 2) >> 1) & 1, dead)) break;
                const int rows = pc.t.n_tok * g;
#pragma unroll 1
                for (int row = (warp - 18) * 32 + lane; row < AR_ROWS; row += 64) {
                    const int place = pc.t.first + row / g;
                    const int token = row < rows ? (a.plan.items ? a.plan.items[place] : place) : -1;
                    const int pos = token >= 0 ? a.positions[token] : -1;
                    const bf16* q = (const bf16*)a.q + (size_t)(pos >= 0 ? token : 0) * a.q_stride + (size_t)(pos >= 0 ? pc.head * g + row % g : 0) * d;
                    float mul = 1.f, fac = a.scale_log2;
                    if (HALF) {
                        // a power of two that brings the row's largest element to [2^14, 2^15)
                        uint32_t amax = 0;
#pragma unroll
                        for (int c = 0; c < DP / 8; ++c) {
                            if (pos < 0 || 8 * c >= d) continue;
                            const uint4 u = __ldg(reinterpret_cast<const uint4*>(q) + c);
                            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) amax = max(amax, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
                        }
                        const int ex = min(max((int)(amax >> 7) - 127, -100), 127);
                        mul = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
                        fac = ldexpf(a.scale_log2, ex - 14);
                    }
                    const uint32_t dst = sQ + (k & 1) * Q_BUF + row * 128, swz = (uint32_t)(row & 7) << 4;
#pragma unroll
                    for (int c = 0; c < DP / 8; ++c) {
                        uint4 u = make_uint4(0u, 0u, 0u, 0u);
                        if (pos >= 0 && 8 * c < d) u = __ldg(reinterpret_cast<const uint4*>(q) + c);
                        if (HALF) {
                            uint32_t* w = &u.x;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const __half2 h = __floats2half2_rn(__uint_as_float(w[j] << 16) * mul, __uint_as_float(w[j] & 0xffff0000u) * mul);
                                w[j] = *reinterpret_cast<const uint32_t*>(&h);
                            }
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n"
                                     ::"r"(dst + (c >> 3) * Q_BLK + (((uint32_t)(c & 7) << 4) ^ swz)), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
                    }
                    s_rows[k & 1].pos[row] = pos;
                    s_rows[k & 1].token[row] = token;
                    s_rows[k & 1].fac[row] = fac;
                }
                tc_fence_async_smem();
                __syncwarp();
                if (lane == 0) rt_mbar_arrive(tc_smem(&s_qbar[0][k & 1]));
            }
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(RT_REGS_OTHER));
        // ---- two warps per group bring its keys (which = 0), two its values: 32 rows of every tile each
        const int w8 = warp - 8, wg = w8 & 1, which = (w8 >> 1) & 1, half = w8 >> 2, row = half * 32 + lane;
        const uint32_t mb_full = bar(wg, M_FULL + which * 2), mb_free = bar(wg, M_FREE + which * 2), mb_meta = bar(wg, M_META);
        const uint32_t buf0 = buf_of(wg, which, 0) + half * 32 * 128;
        RtMeta& meta = s_meta[wg];
        constexpr uint32_t NONE = 0xffffffffu;
        const uint32_t to_values = (uint32_t)a.kv.nkv * a.kv.page_size;
        uint32_t n = 0;                  // this group's tiles so far
        RowWalk walk = s_walk;
        RowPiece pc;
        RtKeys keys;
        keys.n = 0;
        const int* bt = nullptr;
        int i = wg;                      // the next tile of the piece
        bool have = true;
        uint32_t at = NONE;              // its keys' row of this thread, looked up a tile ahead of the loads
        bool hole = false;               // a key that a row may see has no page
        auto look = [&]() {
            while (i >= keys.n) {
                if (!walk.next(a.plan, pc)) { have = false; return; }
                keys = rt_keys(pc);
                const int seq = pc.t.seq >= 0 ? pc.t.seq : a.seq_of_token[a.plan.items[pc.t.first]];
                bt = a.kv.table + (size_t)a.slots[seq] * a.kv.max_pages;
                i = wg;
            }
            const int key = keys.k0 + TC_BN * i + row;
            at = NONE;
            hole = false;
            if (key >= pc.t.key_lo && key < keys.k_end) {
                const int index = a.kv.page_index(key);
                const int page = index < a.kv.max_pages ? __ldg(bt + index) : -1;
                hole = (unsigned)page >= (unsigned)a.kv.num_pages;
                if (!hole) at = a.kv.row0(page, 0, pc.head) + a.kv.offset(key, index);
            }
            i += 2;
        };
        // Scales and marks of a tile, into the place of its turn.  RT_META places: the tile four before has been read when this one's
        // buffer is free, because S of the tile two before was issued after the softmax threads were done with the one before that.
        auto put_meta = [&](float ks, float vs, uint32_t row_at, bool no_page) {
            const int x = n & (RT_META - 1);
            if (which == 0) {
                // (a value row that is not finite has the scale NaN: with the key's it reaches those who see the key and nobody else)
                if (HALF) meta.ks[x][row] = isnan(vs) ? vs : ks;
                const uint32_t seen = __ballot_sync(0xffffffffu, row_at != NONE);
                if (lane == 0) meta.seen[x][half] = seen;
                if (no_page) *a.kv.status = 1;
            } else if (HALF) {
                vs = isnan(vs) ? 0.f : vs;
                meta.vs[x][row] = vs;
                const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(vs));
                if (lane == 0) meta.vmax[x][half] = __uint_as_float(most);
            }
        };
        auto landed = [&](uint32_t x) {
            tc_fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                rt_mbar_arrive(mb_full + 8 * (x & 1));
                if (HALF || which == 0) rt_mbar_arrive(mb_meta + 8 * (x & (RT_META - 1)));
            }
        };
        auto wait_free = [&]() -> bool { return n < 2 || tc_wait_warp(mb_free + 8 * (n & 1), ((n - 2) >> 1) & 1, dead); };
        look();
        const unsigned char* pool = a.kv.pool;
        if constexpr (HALF) {
            // NP neighbouring lanes read a row, 16 bytes each: load j has rows j RI .. j RI + RI - 1 of the warp's 32
            constexpr int NP = DP / 16, RI = 32 / NP;
            const int p = lane % NP, rl = lane / NP;
            const bool in = 16 * p < d;
            uint4 data[NP];
            float ks = 0.f, vs = 0.f;
            auto load = [&](int j) {
                const uint32_t r = __shfl_sync(0xffffffffu, at, j * RI + rl);
                data[j] = in && r != NONE ? __ldg(reinterpret_cast<const uint4*>(pool + (size_t)(which ? r + to_values : r) * d) + p)
                                          : make_uint4(0u, 0u, 0u, 0u);
            };
            auto load_scales = [&]() {
                ks = which == 0 && at != NONE ? __ldg(a.kv.scales + at) : 0.f;
                vs = at != NONE ? __ldg(a.kv.scales + at + to_values) : 0.f;
            };
            if (have) {
                load_scales();
#pragma unroll
                for (int j = 0; j < NP; ++j) load(j);
            }
            while (have) {
                const uint32_t mine = at;
                const bool no_page = hole;
                look();                                      // `at`: the next tile's (NONE behind the last one)
                if (!have) at = NONE;
                if (!wait_free()) break;
                const uint32_t buf = buf0 + (n & 1) * BUF + (p >> 2) * KV_BLK;
                put_meta(ks, vs, mine, no_page);
                load_scales();
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    uint32_t h[8];
                    c8_halves<FORM>(data[j].x, h[0], h[1]);
                    c8_halves<FORM>(data[j].y, h[2], h[3]);
                    c8_halves<FORM>(data[j].z, h[4], h[5]);
                    c8_halves<FORM>(data[j].w, h[6], h[7]);
                    load(j);                                 // the next tile's, as soon as the registers are free
                    const uint32_t r = j * RI + rl;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {            // eight dimensions each; the upper half of a row the other way round (banks)
                        const bool flip = (p >> 2) & 1;
                        const uint32_t c = (2 * p + (flip ? 1 - k : k)) & 7;
                        const bool hi = flip ? k == 0 : k == 1;
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n"
                                     ::"r"(buf + r * 128 + ((c ^ (r & 7)) << 4)), "r"(hi ? h[4] : h[0]), "r"(hi ? h[5] : h[1]),
                                       "r"(hi ? h[6] : h[2]), "r"(hi ? h[7] : h[3]) : "memory");
                    }
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
                if (!wait_free()) { alive = false; break; }
                const uint32_t buf = buf0 + (n & 1) * BUF + (p >> 3) * KV_BLK;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const int row_j = j * RI + rl;
                    const uint32_t r = __shfl_sync(0xffffffffu, at, row_j);
                    const bool ok = in && r != NONE;
                    tc_cp16(buf + row_j * 128 + (((p & 7) ^ (row_j & 7)) << 4),
                            ok ? pool + (size_t)(which ? r + to_values : r) * d * 2 + 16 * p : pool, ok);
                }
                tc_cp_commit();
                put_meta(0.f, 0.f, at, hole);
                ++n;
                look();
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
        const int wg = warp >> 2, row = tid & 127, warp4 = warp & 3;
        const uint32_t t_wg = tmem + wg * WG_COLS + ((uint32_t)(warp4 * 32) << 16);
        const uint32_t mb_s = bar(wg, M_S), mb_o = bar(wg, M_O), mb_meta = bar(wg, M_META);
        const RtMeta& meta = s_meta[wg];
        bool alive = true;
        uint32_t n = 0;                                  // tiles of this group so far
        RowWalk walk = s_walk;
        RowPiece pc;
        int k = 0;
        for (; walk.next(a.plan, pc); ++k) {
            const RtKeys keys = rt_keys(pc);
            const int mine = rt_share(keys.n, wg), rows = pc.t.n_tok * g;
            const int head = pc.head * g + row % g;
            if (alive) alive = tc_wait_warp(tc_smem(&s_qbar[0][k & 1]), (k >> 1) & 1, dead);
            const int pos = s_rows[k & 1].pos[row], token = s_rows[k & 1].token[row];
            const float fac = s_rows[k & 1].fac[row];
            __syncwarp();
            if (lane == 0) rt_mbar_arrive(tc_smem(&s_qbar[1][k & 1]));
            if (wg == 1 && k > 0) rt_taken_sync();       // the first group has read this one's O of the piece before
            const int hi = min(pos + 1, keys.k_end);
            const int lo = max(pc.t.key_lo, a.window > 0 ? pos - a.window + 1 : 0);
            float ref = -INFINITY, sum = 0.f;
            for (int i = 0; i < mine; ++i) {
                const uint32_t x = n + i;
                const int key0 = keys.k0 + TC_BN * (wg + 2 * i), mt = x & (RT_META - 1);
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
                uint32_t w[TC_BN / 2];
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
                        const __nv_bfloat162 h0 = __floats2bfloat162_rn(p[0], p[1]), h1 = __floats2bfloat162_rn(p[2], p[3]);
                        w[c / 2] = *reinterpret_cast<const uint32_t*>(&h0);
                        w[c / 2 + 1] = *reinterpret_cast<const uint32_t*>(&h1);
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
                sum += ((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7]));
                tc_st_wait();
                tc_fence_before_sync();
                if (alive) rt_arrive(wg, 1);
                else rt_sync(wg, 1);
            }
            if (mine > 0) {
                if (alive) alive = tc_wait_warp(mb_o, (n + mine - 1) & 1, dead);
                tc_fence_after_sync();
            }
            n += mine;
            // ---- the groups' sums
            if (wg == 1) {
                s_mrg[0][row] = mine > 0 ? ref : -INFINITY;
                s_mrg[1][row] = sum;
                tc_fence_before_sync();
                rt_share_arrive();
            } else {
                rt_share_sync();
                tc_fence_after_sync();
                const bool two = keys.n > 1;             // the second group has tiles
                const float r1 = s_mrg[0][row], m = fmaxf(ref, r1);
                const float a0 = ar_weight(ref, m), a1 = ar_weight(r1, m);
                const float l = sum * a0 + s_mrg[1][row] * a1;
                const bool direct = a.direct && pc.whole, mine_to_store = row < rows && pos >= 0 && alive;
                const size_t slot = ((size_t)(pc.unit + blockIdx.x)) * AR_ROWS + row;
                if (!direct && row < rows) { a.parts.r[slot] = m; a.parts.l[slot] = l; }
                const float inv = l == 0.f ? 0.f : 1.f / l;
                bf16* out = (bf16*)a.out + ((size_t)(token >= 0 ? token : 0) * a.plan.nh + head) * d;
                float* part = a.parts.o + slot * d;
#pragma unroll
                for (int cb = 0; cb < DP / 16; ++cb) {
                    float o[16], o1[16];
                    uint32_t* r0 = reinterpret_cast<uint32_t*>(o);
                    uint32_t* r1p = reinterpret_cast<uint32_t*>(o1);
                    const uint32_t t0 = t_wg + T_O + cb * 16, t1 = t0 + WG_COLS;
#define RT_LD16(r, t)                                                                                                              \
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"         \
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),     \
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(t) : "memory")
                    __syncwarp();
                    RT_LD16(r0, t0);
                    if (two) RT_LD16(r1p, t1);
                    tc_ld_wait();
                    if (cb * 16 >= d) continue;
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = o[e] * a0 + (two ? o1[e] * a1 : 0.f);
                    if (mine_to_store && direct) {
#pragma unroll
                        for (int e = 0; e < 16; e += 8) {
                            uint32_t h[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const __nv_bfloat162 b = __floats2bfloat162_rn(o[e + 2 * j] * inv, o[e + 2 * j + 1] * inv);
                                h[j] = *reinterpret_cast<const uint32_t*>(&b);
                            }
                            *reinterpret_cast<uint4*>(out + cb * 16 + e) = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                    } else if (mine_to_store) {
#pragma unroll
                        for (int e = 0; e < 16; e += 4) store4(part + cb * 16 + e, make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]));
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                rt_taken_arrive();
            }
        }
        if (wg == 1 && k > 0) rt_taken_sync();
    }
    tc_fence_before_sync();
    asm volatile("bar.sync 7, %0;\n" ::"n"(RT_THREADS) : "memory");
    if (s_dead && tid == 0) atomicExch(a.kv.status, 3);
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}

template <int FORM, int DP> static int rt_run(const RowArgs& a, cudaStream_t s) {
    constexpr size_t smem = 2 * (DP / 64) * TC_BM * 128 + 8 * (DP / 64) * TC_BN * 128 + 1024;
    auto kernel = attention_rows_tc_kernel<FORM, DP>;
    AR_ALLOW_SMEM(kernel, smem);
    // the redistribution of registers moves what the launch got, and waits for more for ever: only for a kernel compiled as assumed
    static int regs[64] = {0};
    int& have = regs[ar_device()];
    if (!have) {
        cudaFuncAttributes attr;
        const cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
        if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
        have = attr.numRegs;
    }
    if (have * RT_THREADS < 256 * RT_REGS_SOFTMAX + 384 * RT_REGS_OTHER) return ST_ERR_TOO_LARGE;
    kernel<<<a.plan.ctas, RT_THREADS, smem, s>>>(a);
    return st_launch_status();
}

int ar_rows_tc(const RowArgs& a, int form, cudaStream_t s) {
    if (form == C8_INT8) return a.d <= 64 ? rt_run<C8_INT8, 64>(a, s) : rt_run<C8_INT8, 128>(a, s);
    if (form == C8_E4M3) return a.d <= 64 ? rt_run<C8_E4M3, 64>(a, s) : rt_run<C8_E4M3, 128>(a, s);
    return a.d <= 64 ? rt_run<C8_BF16, 64>(a, s) : rt_run<C8_BF16, 128>(a, s);
}
