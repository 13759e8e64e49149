// cw_tree_tc.cu -- cw_tree_attention over 16-bit caches on the 5th-generation
// tensor cores (tcgen05, operands staged by TMA, accumulators in TMEM), for more rows
// than cw_tree_few.cu takes.
//
// Per 64-key tile and 128 query rows (one TMEM lane a row):
//
//   S [128 x 64]  = Q K^T   both from shared memory (128-byte swizzled)
//   P [128 x 64]  = 2^(c S - ref), rounded to the type, over S's own columns
//   O [128 x D]  += P V     P from TMEM, V as it lies in memory (keys x dims)
//
// The cache is read once: all G query heads of a kv head and all nodes of the
// request share a tile (up to 128 rows, or 256 with two row blocks per CTA; at 256
// dims 128, whose second block reads the tile through L2).  A tile of 64 keys at
// D = 128 is 32 KB, 0.75 us of an SM's share of the memory bandwidth.  128 rows take
// about as long (two CTAs per SM: 32 x 32 nodes at 8192 in 162 us, memory alone 109).
// 256 rows are bound by their exponentials and the issue slots around them: 1.4 us a
// tile, of which 0.6 us are the special-function unit's alone (2 x 64 nodes at 131000
// in 360 us, 309 in a short run; memory alone 151).
//
// Warps: 4 (or 2 x 4) softmax warps, a thread per row, so row maxima and sums need
// no exchange; one TMA warp; one elected MMA lane.  S has two TMEM buffers: the scores of
// tile i + 1 are formed while the weights of tile i are.  O is rescaled only when a
// row's maximum has grown by 2^8 since its last reference (weights then stay below 2^8,
// in f16 2^15, inside both types); the final division makes the reference drop out.
// Weights are rounded to the cache's type for the second product; the row's sum is
// taken over the rounded weights, so a constant v comes out exact.
//
// Keys that not every row sees lie in the tiles of the nodes, the last tile and,
// with a window, those at its edge.  There each thread forms its row's 64-bit set
// of seen keys, v rows past the end are zeroed, and a tile whose v holds values
// that are not finite is mended: those values are taken out of the product and
// added to the rows that see them.  Keys without a page (an id outside the cache) are
// zeros in shared memory, and once there is one the threads look ids up and mask them.
#include <algorithm>
#include <mutex>

#include "cw_tree_tc.cuh"

namespace cw {

// A parity wait tells a phase from the one before it only, so a barrier that is
// waited on once per tile is doubled by tile parity: when tile n - 1's phase is
// waited for, tile n - 3's is known to be over (scores of tile n - 1 come after it).
struct TtBars {
    uint64_t full[TT_STAGES], empty[TT_STAGES];
    uint64_t q_full[2], s_full[2][2], p_full[2][2], pv[2][2], done;  // [row block][tile % 2]
    uint32_t tmem, failed, lost;  // lost: some key has no page
    TreeShared run;
};

// Barrier and OR over the threads of the item's active row blocks (one named barrier
// for each count: a block may run ahead through items that are not its own).
__device__ __forceinline__ bool tt_any(bool x, int blocks) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)x), "r"(blocks), "r"(blocks * 128)
        : "memory");
    return r != 0;
}

// Which of the keys [j0, j1) have a page (out of line: 16 x 100 nodes of 64 dims at 4500
// take 100.6 us, 103.5 with the loop in its place).
__device__ __noinline__ uint64_t tt_have(const TreeArgs& a, int r, int j0, int j1) {
    uint64_t have = 0;
    for (int j = j0; j < j1; j++) have |= (uint64_t)tree_has(a, r, j) << (j - j0);
    return have;
}

// The shapes of one instance.  HD: head dims rounded up; a thread's keys of a tile
// are KEYS consecutive ones, so SPLIT lanes share a row.
template <int HD, int NB, int SPLIT> struct TtShape {
    static constexpr int COLS = HD / 64;                // 64-element column blocks
    static constexpr int STAGE = COLS * TR_TILE * 128;  // a tile of 64 keys
    // TMEM of a row block: two buffers of scores, then O.  (128-key tiles with one buffer,
    // half the hand-overs per key, were slower: the scores of the next tile then wait for
    // the product of this one; 32 x 32 nodes at 8192: 209 us against 176.)
    static constexpr int TCOLS = 2 * TR_TILE + HD;
    static constexpr uint32_t TMEM = NB * TCOLS <= 256 ? 256 : 512;
    static constexpr int THREADS = NB * 128 + 64;
    static constexpr int PER_SM = NB == 1 && HD <= 128 ? 2 : 1;
    static constexpr int KEYS = TR_TILE / SPLIT;
    static constexpr int LANES = 128 / SPLIT;           // rows of a row block
};

template <bool BF, int HD, int NB, int SPLIT>
__global__ void __launch_bounds__(NB * 128 + 64, TtShape<HD, NB, SPLIT>::PER_SM)
    k_tree_tc(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
              const __grid_constant__ TreeArgs a, int stages, int q_rows) {
    typedef TtShape<HD, NB, SPLIT> Z;
    constexpr int COLS = Z::COLS, TILE = TR_TILE, SB = 2;
    constexpr int STAGE = Z::STAGE, TCOLS = Z::TCOLS, KEYS = Z::KEYS, LANES = Z::LANES;
    static_assert(NB == 1 || SPLIT == 1, "a split row block is the only one");
    extern __shared__ __align__(1024) uint8_t sm[];
    const int q_block = q_rows * 128;         // bytes of a column block of the queries
    uint8_t* s_q = sm;                        // [NB][COLS][q_rows][128]
    uint8_t* ring = sm + NB * COLS * q_block;
    TtBars* bars = (TtBars*)(ring + stages * STAGE);
    // reference and sum of each lane's part of a row, when the queries are done with
    float2* s_ml = HD > 64 ? (float2*)(s_q + 128 * 128) : (float2*)(bars + 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // the swizzle counts from 1024-byte boundaries; no static shared memory precedes
    if (smem_addr(sm) & 1023) {
        if (tid == 0) tree_bad(a);
        return;
    }
    if (warp == 0) tmem_alloc(&bars->tmem, Z::TMEM);
    if (tid == 32) {
        for (int s = 0; s < stages; s++) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int b = 0; b < NB; b++) {
            mbar_init(&bars->q_full[b], 4);
            for (int i = 0; i < 2; i++) {
                mbar_init(&bars->pv[b][i], 1);
                mbar_init(&bars->s_full[b][i], 1);
                mbar_init(&bars->p_full[b][i], 4);
            }
        }
        mbar_init(&bars->done, 1);
        bars->failed = bars->lost = 0;
        fence_mbar_init();
    }
    pdl_wait();  // the setup above overlaps the launch before
    pdl_trigger();
    TreeRun run = tree_run<Z::THREADS>(a, &bars->run);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return tt_wait(bar, parity, &bars->failed, a.status);
    };
    auto all = [&](uint64_t* bar, uint32_t parity) {  // the same answer for the warp
        return __all_sync(FULL, wait(bar, parity)) != 0;
    };
    TreeItem it;
    bool any = false, ok = true;
    const bool wide = tt_wide(a.D);
    const TtTile tile = wide ? TtTile{COLS * 1024, 1024} : TtTile{1024, TILE * 128};
    TtPlace at = {0, 0};

    if (warp == NB * 4) {  // ---- TMA: all lanes, a box each
        TtFeed<COLS, TILE> feed(a, ring, bars->full, bars->empty, &bars->lost, stages, tile);
        if (lane == 0) {
            tma_prefetch_desc(&map_k);
            tma_prefetch_desc(&map_v);
        }
        while (run.left > 0 && ok) {
            it = tree_next(a, run);
            feed.begin(it);
            int now = feed.place(0);
            ok = feed.load(&map_k, now, all);
            for (int i = 0; i < it.tiles && ok; i++) {
                const int next = feed.place(i + 1);
                if (i + 1 < it.tiles) ok = feed.load(&map_k, next, all);
                ok = ok && feed.load(&map_v, now, all);
                now = next;
            }
        }
        if (!ok) feed.drain();
    } else if (warp == NB * 4 + 1) {  // ---- MMA: one elected lane
        constexpr uint32_t id_s = tt_idesc<BF>(TILE, false, false);
        constexpr uint32_t id_o = tt_idesc<BF>(HD, false, true);
        const uint64_t q0 = umma_desc_sw128(smem_addr(s_q)), kv0 = tt_desc(smem_addr(ring), tile);
        const int steps = (a.D + 15) / 16;
        if (tt_elect()) {
        uint32_t n[2] = {0, 0}, items[2] = {0, 0};  // tiles and items of each row block
        while (run.left > 0 && ok) {
            it = tree_next(a, run);
            const int blocks = it.rows > 128 ? NB : 1;
            for (int b = 0; b < blocks && ok; b++) ok = wait(&bars->q_full[b], items[b]++);
            // S = Q K^T of tile i, of each row block
            auto scores = [&](int i) {
                const int s = at.stage;
                ok = ok && wait(&bars->full[s], at.phase);
                at.next(stages);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    if (b >= blocks) break;
                    const uint32_t m = n[b] + i;
                    // this buffer's weights went into the product of tile i - 2
                    if (i >= 2) ok = ok && wait(&bars->pv[b][m & 1], (m - 2) >> 1);
                    tc_fence_after();
                    if (ok) {
                        const uint32_t d = tmem + b * TCOLS + (m & 1) * TILE;
                        const uint64_t dq = q0 + ((b * COLS * q_block) >> 4),
                                       dk = kv0 + ((s * STAGE) >> 4);
#pragma unroll
                        for (int x = 0; x < HD / 16; x++)
                            if (x < steps)
                                umma_f16(d, dq + (((x >> 2) * q_block + (x & 3) * 32) >> 4),
                                         dk + (((x >> 2) * tile.col + (x & 3) * 32) >> 4), id_s,
                                         x > 0);
                        tc_commit(&bars->s_full[b][m & 1]);
                        if (b + 1 == blocks) tc_commit(&bars->empty[s]);
                    }
                }
            };
            scores(0);
            for (int i = 0; i < it.tiles && ok; i++) {
                if (i + 1 < it.tiles) scores(i + 1);
                // O += P V of tile i
                const int s = at.stage;
                ok = ok && wait(&bars->full[s], at.phase);
                at.next(stages);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    if (b >= blocks) break;
                    const uint32_t m = n[b] + i;
                    ok = ok && wait(&bars->p_full[b][m & 1], m >> 1);
                    tc_fence_after();
                    if (ok) {
                        const uint32_t p = tmem + b * TCOLS + (m & 1) * TILE;
                        const uint64_t dv = kv0 + ((s * STAGE) >> 4);
                        // 16 keys go to the lanes that weigh them
#pragma unroll
                        for (int x = 0; x < TILE / 16; x++) {
                            auto off = [&](int quad) {
                                return x * 16 / KEYS == quad * 32 / LANES ? 0u : ~0u;
                            };
                            tt_mma_ts(tmem + b * TCOLS + SB * TILE, p + 8 * x,
                                      dv + ((x * 2 * tile.group) >> 4), id_o, off(0), off(1),
                                      off(2), off(3));
                        }
                        tc_commit(&bars->pv[b][m & 1]);
                        if (b + 1 == blocks) tc_commit(&bars->empty[s]);
                    }
                }
            }
            for (int b = 0; b < blocks; b++) n[b] += it.tiles;
        }
        // every product issued has ended before the block frees its TMEM
        tc_commit(&bars->done);
        (void)mbar_wait(&bars->done, 0, TT_WAIT_NS);
        }
        __syncwarp();
    } else {  // ---- softmax: a thread per row and part of the keys
        // lane m weighs keys [part * KEYS, ..+KEYS) of each tile for row r
        const int b = warp >> 2, m = tid & 127, r = m % LANES, part = m / LANES;
        const uint32_t lanes = tmem + b * TCOLS + ((uint32_t)(warp & 3) << 21);
        const uint32_t t_o = lanes + SB * TILE;
        uint32_t n = 0;
        const float log2e = 1.44269504088896341f;
        const bool cap = a.softcap > 0.f;
        const float c2 = cap ? log2e : a.scale * log2e;
        const float y2 = cap ? 2.f * log2e * a.scale / a.softcap : 0.f;
        // a score with the cap: tanh(y) = 1 - 2 / (1 + e^2y), off by 2^-22, times
        // softcap far below one rounding of the weight
        auto capped = [&](float s) {
            const float y = s * y2;
            return a.softcap - __fdividef(2.f * a.softcap, 1.f + tt_exp2(y > 120.f ? 120.f : y));
        };
        uint8_t* q_sm = s_q + b * COLS * q_block;
        while (run.left > 0) {
            it = tree_next(a, run);
            any = true;
            const int blocks = it.rows > 128 ? NB : 1;
            const int tiles = it.tiles;
            TtPlace at_v = at;  // of the item's first V tile
            at_v.skip(tiles > 1 ? 2 : 1, stages);
            at.skip(2 * tiles % (2 * stages), stages);
            if (b >= blocks) continue;
            const int m0 = it.block * a.bm + b * 128;       // row 0 of the request's rows
            const int rows = min(it.rows - b * 128, 128);
            const bool work = (warp & 3) * 32 % LANES < rows;  // the warp has rows
            const int key0 = (it.q.tile0 + it.tile) * TR_TILE;
            const int end = min(it.q.keys, key0 + it.tiles * TR_TILE);  // of this piece's keys
            // ---- queries, and this row's window
            for (int i = m; i < rows * COLS * 8; i += 128) {
                const int qr = i / (COLS * 8), c = i % (COLS * 8);
                const int node = (m0 + qr) / a.G, gi = (m0 + qr) - node * a.G;
                uint4 x = make_uint4(0, 0, 0, 0);
                if (c * 8 < a.D)
                    x = *(const uint4*)((const uint16_t*)a.q +
                                        (long long)(it.q.row0 + node) * a.q_stride +
                                        (long long)(it.head * a.G + gi) * a.D + c * 8);
#pragma unroll
                for (int s = 0; s < SPLIT; s++)  // once for each part's lanes
                    *(uint4*)(q_sm + (c >> 3) * q_block + (qr + s * LANES) * 128 +
                              (((c & 7) ^ (qr & 7)) << 4)) = x;
            }
            int edge = 0, edge_max = 0;  // this row's, and the largest of the item's rows
            if (a.window > 0) {
                if (r < rows) edge = tree_edge(a, it.q, m0 + r);
                const int last = (it.block * a.bm + it.rows - 1) / a.G;
                for (int node = it.block * a.bm / a.G + lane; node <= last; node += 32)
                    edge_max = max(edge_max, tree_edge(a, it.q, node * a.G));
                edge_max = __reduce_max_sync(FULL, edge_max);
            }
            if (work) {
                uint32_t z[32];
#pragma unroll
                for (int i = 0; i < 32; i++) z[i] = 0;
#pragma unroll
                for (int c = 0; c < HD; c += 32) tt_st32(t_o + c, z);
                tt_wait_st();
            }
            tt_fence_async();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->q_full[b]);
            // running maximum of the scores, the weights' reference (in powers of two),
            // and the sum of the weights
            float top = -INFINITY, ref = -INFINITY, sum = 0.f;
            for (int i = 0; i < tiles; i++, n++) {
                const int kt = key0 + i * TILE;
                const bool mixed = kt + TILE > end || kt + TILE > it.q.len || kt < edge_max;
                uint64_t sees = ~0ull;  // this row's, of the tile's keys
                if (mixed && (kt < edge || kt + TILE > it.q.len || kt + TILE > end))
                    sees = r < rows ? tree_sees(a, it.q, m0 + r, kt) : 0;
                wait(&bars->s_full[b][n & 1], n >> 1);
                __syncwarp();
                tc_fence_after();
                // set before the tile's keys were, if one of them has no page
                const bool lost = *(volatile uint32_t*)&bars->lost;
                const uint32_t t_s = lanes + (n & 1) * TILE;
                if (work) {
                    float s[KEYS];
                    tt_load<KEYS>(t_s + part * KEYS, (uint32_t*)s);
                    if (cap) {
#pragma unroll
                        for (int j = 0; j < KEYS; j++) s[j] = capped(s[j]);
                    }
                    if (mixed || lost) {
                        uint64_t mine = sees >> (part * KEYS);
                        if (lost) {
                            const int j0 = kt + part * KEYS;
                            mine &= tt_have(a, it.r, j0, min(end, j0 + KEYS));
                        }
#pragma unroll
                        for (int j = 0; j < KEYS; j++)
                            if (!(mine >> j & 1)) s[j] = -INFINITY;
                    }
                    float t0 = top, t1 = top, t2 = top, t3 = top;
#pragma unroll
                    for (int j = 0; j < KEYS; j += 4) {
                        t0 = fmaxf(t0, s[j]);
                        t1 = fmaxf(t1, s[j + 1]);
                        t2 = fmaxf(t2, s[j + 2]);
                        t3 = fmaxf(t3, s[j + 3]);
                    }
                    top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
                    const float want = top == -INFINITY ? -INFINITY : top * c2 - TT_LIFT<BF>;
                    if (i == 0) {
                        ref = want;
                    } else if (__any_sync(FULL, r < rows && want - ref > 8.f)) {
                        const float fix = ref == -INFINITY ? 0.f : tt_exp2(ref - want);
                        wait(&bars->pv[b][(n - 1) & 1], (n - 1) >> 1);  // O: the tiles so far
                        __syncwarp();
                        tc_fence_after();
                        sum *= fix;
                        ref = want;
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tt_load<32>(t_o + c, o);
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                o[j] = __float_as_uint(__uint_as_float(o[j]) * fix);
                            tt_st32(t_o + c, o);
                        }
                    }
                    const float from = ref == -INFINITY ? 0.f : ref;
                    float l0 = 0.f, l1 = 0.f;
                    uint32_t p[KEYS / 2];
#pragma unroll
                    for (int j = 0; j < KEYS; j++) s[j] = tt_exp2(fmaf(s[j], c2, -from));
#pragma unroll
                    for (int j = 0; j < KEYS / 2; j += 2) {
                        p[j] = tt_pack<BF>(s[2 * j], s[2 * j + 1], l0);
                        p[j + 1] = tt_pack<BF>(s[2 * j + 2], s[2 * j + 3], l1);
                    }
                    sum += l0 + l1;
                    tt_st<KEYS / 2>(t_s + part * (KEYS / 2), p);
                    tt_wait_st();
                }
                if (mixed) {  // v rows past the end, and values that are not finite
                    wait(&bars->full[at_v.stage], at_v.phase);
                    __syncwarp();
                    uint8_t* v = ring + at_v.stage * STAGE;
                    auto chunk = [&](int j, int c) { return v + tile.at(j, c); };
                    const int live = end - kt;
                    bool odd = false;
                    for (int x = b * 128 + m; x < COLS * TILE * 8; x += blocks * 128) {
                        uint4* w = (uint4*)chunk(x / (COLS * 8), x % (COLS * 8));
                        if (x / (COLS * 8) >= live) *w = make_uint4(0, 0, 0, 0);
                        else odd |= tt_odd8<BF>(*w);
                    }
                    if (tt_any(odd, blocks)) {
                        if (work) {
                            if (i > 0) wait(&bars->pv[b][(n - 1) & 1], (n - 1) >> 1);
                            __syncwarp();
                            tc_fence_after();
#pragma unroll 1
                            for (int j = 0; j < min(live, TILE); j++)
#pragma unroll 1
                                for (int c = 0; c < COLS * 8; c++) {
                                    const uint4 x = *(const uint4*)chunk(j, c);
                                    if (!tt_odd8<BF>(x)) continue;
#pragma unroll 1
                                    for (int e = 0; e < 8; e++) {
                                        const uint32_t bits = ((const uint16_t*)chunk(j, c))[e];
                                        if (!tt_odd<BF>(bits)) continue;
                                        uint32_t pj = tt_ld1(t_s + (j >> 1));
                                        uint32_t oj = tt_ld1(t_o + c * 8 + e);
                                        asm volatile("tcgen05.wait::ld.sync.aligned;"
                                                     : "+r"(pj), "+r"(oj)::"memory");
                                        float o = __uint_as_float(oj);
                                        if ((sees >> j & 1) && j / KEYS == part)
                                            o = fmaf(tt_value<BF>(j & 1 ? pj >> 16 : pj & 0xffffu),
                                                     tt_value<BF>(bits), o);
                                        __syncwarp();
                                        tt_st1(t_o + c * 8 + e, __float_as_uint(o));
                                        tt_wait_st();
                                    }
                                }
                        }
                        (void)tt_any(false, blocks);  // all have read them
                        for (int x = b * 128 + m; x < COLS * TILE * 8; x += blocks * 128) {
                            uint16_t* w = (uint16_t*)chunk(x / (COLS * 8), x % (COLS * 8));
                            for (int e = 0; e < 8; e++)
                                if (tt_odd<BF>(w[e])) w[e] = 0;
                        }
                    }
                    tt_fence_async();
                    // both row blocks read the mended tile
                    if (NB > 1) (void)tt_any(false, blocks);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->p_full[b][n & 1]);
                at_v.skip(i + 2 < tiles ? 2 : 1, stages);
            }
            // ---- the item's end
            wait(&bars->pv[b][(n - 1) & 1], (n - 1) >> 1);
            __syncwarp();
            tc_fence_after();
            const size_t piece =
                ((size_t)blockIdx.x * 2 + tree_slot(run, it)) * a.bm + b * 128 + r;
            const int node = (m0 + r) / a.G, gi = (m0 + r) - node * a.G;
            uint16_t* out = (uint16_t*)a.out +
                            ((long long)(it.q.row0 + node) * a.H + it.head * a.G + gi) * a.D;
            // N f32 sums of columns c.. of this row: the result, or the partial state
            auto put = [&](const float* o, int c, float inv) {
                if (it.whole) {
                    float unused = 0.f;
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        w[e] = inv == 0.f ? 0u : tt_pack<BF>(o[2 * e] * inv, o[2 * e + 1] * inv, unused);
                    *(uint4*)(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    *(float4*)(a.part + piece * a.dp + c) = make_float4(o[0], o[1], o[2], o[3]);
                    *(float4*)(a.part + piece * a.dp + c + 4) = make_float4(o[4], o[5], o[6], o[7]);
                }
            };
            if constexpr (SPLIT == 1) {
                const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
                if (r < rows && !it.whole) a.ml[piece] = make_float2(ref, sum);
                if (work) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
                        __syncwarp();
                        tt_load<32>(t_o + c, (uint32_t*)o);
#pragma unroll
                        for (int j = 0; j < 32; j += 8)
                            if (r < rows && c + j < a.D) put(o + j, c + j, inv);
                    }
                }
            } else {
                // join the SPLIT parts of each row: 32 columns at a time through the
                // queries' place, 16-byte chunks exclusive-ored with the lane
                s_ml[m] = make_float2(ref, sum);
                (void)tt_any(false, 1);
                float top = -INFINITY, l = 0.f;
#pragma unroll
                for (int s = 0; s < SPLIT; s++) top = fmaxf(top, s_ml[s * LANES + r].x);
#pragma unroll
                for (int s = 0; s < SPLIT; s++) {
                    const float2 x = s_ml[s * LANES + r];
                    if (x.y != 0.f) l += x.y * tt_exp2(x.x - top);  // NaN stays
                }
                const float own = ref == -INFINITY ? 0.f : tt_exp2(ref - top);
                const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
                if (r < rows && part == 0 && !it.whole) a.ml[piece] = make_float2(top, l);
#pragma unroll 1
                for (int c = 0; c < HD && c < a.D; c += 32) {
                    if (work) {
                        float o[32];
                        tt_load<32>(t_o + c, (uint32_t*)o);
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            *(float4*)(q_sm + m * 128 + ((j ^ (m & 7)) << 4)) =
                                make_float4(o[4 * j] * own, o[4 * j + 1] * own, o[4 * j + 2] * own,
                                            o[4 * j + 3] * own);
                    }
                    (void)tt_any(false, 1);
                    if (r < rows) {  // this thread: 32 / SPLIT of the columns
#pragma unroll
                        for (int j = 0; j < 8 / SPLIT; j += 2) {
                            const int at = part * (8 / SPLIT) + j;
                            float o[8] = {};
#pragma unroll
                            for (int s = 0; s < SPLIT; s++) {
                                const uint8_t* from = q_sm + (s * LANES + r) * 128;
                                const float4 x = *(const float4*)(from + ((at ^ (r & 7)) << 4));
                                const float4 y = *(const float4*)(from + (((at + 1) ^ (r & 7)) << 4));
                                o[0] += x.x, o[1] += x.y, o[2] += x.z, o[3] += x.w;
                                o[4] += y.x, o[5] += y.y, o[6] += y.z, o[7] += y.w;
                            }
                            if (c + at * 4 < a.D) put(o, c + at * 4, inv);
                        }
                    }
                    (void)tt_any(false, 1);
                }
            }
            tc_fence_before();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0) tree_record(a, run, it, any);
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, Z::TMEM);
    }
}

static PFN_cuTensorMapEncodeTiled_v12000 tt_encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
    });
    return fn;
}

// The cache's rows in groups of 8 (a page holds whole groups): [groups][D / 64][8][64],
// or with a ragged D [groups][1][8][D], whose columns past D read zeros; boxes of one
// page, 64 rows at most.
int tt_map(CUtensorMap* map, const void* base, const TreeArgs& a, bool bf) {
    auto enc = tt_encode_fn();
    CW_CHECK(enc, CW_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const bool wide = tt_wide(a.D);
    cuuint64_t dims[4] = {(cuuint64_t)(wide ? 64 : a.D), 8, (cuuint64_t)(wide ? a.D / 64 : 1),
                          (cuuint64_t)a.n_pages * a.K * a.page / 8};
    cuuint64_t strides[3] = {(cuuint64_t)a.D * 2, 128, (cuuint64_t)a.D * 16};
    cuuint32_t box[4] = {64, 8, (cuuint32_t)dims[2], (cuuint32_t)std::min(a.page, TR_TILE) / 8};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                     const_cast<void*>(base), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CW_CHECK(r == CUDA_SUCCESS, CW_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return CW_OK;
}

// The query rows [n_rows][H][D], boxes of a request's nodes by a kv head's G heads.
int tt_map_q(CUtensorMap* map, const TreeArgs& a, bool bf) {
    auto enc = tt_encode_fn();
    CW_CHECK(enc, CW_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.H, (cuuint64_t)a.n_rows};
    cuuint64_t strides[2] = {(cuuint64_t)a.D * 2,
                             (cuuint64_t)std::max(a.q_stride, (long long)a.H * a.D) * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)a.G, (cuuint32_t)a.max_nodes};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                     const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CW_CHECK(r == CUDA_SUCCESS, CW_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return CW_OK;
}

bool tree_tc_takes(const cw_tree_attn_args& p, const void* q, const void* k, const void* v) {
    const bool pages = p.page_size == 8 || p.page_size == 16 || p.page_size == 32 ||
                       p.page_size % TR_TILE == 0;
    return p.type != CW_GGUF_F32 && p.head_dim % 8 == 0 && pages && p.q_off % 8 == 0 &&
           p.q_stride % 8 == 0 && (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) == 0 &&
           (uint64_t)p.n_pages * p.n_kv * p.page_size < (1ull << 31);
}
// Two row blocks to a CTA where a request can have more than 128 rows, so that its
// keys are still read once (their TMEM, 2 x (128 + 256) columns, does not fit at 256).
int tree_tc_rows(const TreeArgs& a) {
    const int most = a.max_nodes * a.G;
    if (tt_few_takes(a)) return most <= 16 ? 16 : most <= 32 ? 32 : 64;
    return most > 128 && a.D <= 128 ? 256 : 128;
}
static int tt_per_sm(const TreeArgs& a) { return a.bm == 128 && a.D <= 128 ? 2 : 1; }
int tree_tc_grid(cw_ctx* ctx, const TreeArgs& a) { return ctx->sm_count * tt_per_sm(a); }

template <bool BF, int HD, int NB, int SPLIT>
static int tt_go(cw_ctx* ctx, const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv,
                 int grid) {
    auto kern = k_tree_tc<BF, HD, NB, SPLIT>;
    // the ring takes what the queries leave of the SM's shared memory (two CTAs of
    // 113 KB or one of 227 KB); without a split, products read rows past q_rows as
    // whatever follows
    typedef TtShape<HD, NB, SPLIT> Z;
    const int q_rows = SPLIT > 1 ? 128 : std::min(128, (a.max_nodes * a.G + 7) / 8 * 8);
    const size_t q = (size_t)NB * Z::COLS * q_rows * 128, stage = Z::STAGE;
    const size_t cap = Z::PER_SM == 2 ? 115712 : 232448, fixed = sizeof(TtBars) + (HD > 64 ? 0 : 128 * 8);
    const int stages = (int)std::min<size_t>((cap - fixed - q) / stage, TT_STAGES);
    const size_t smem = fixed + q + stages * stage;
    static bool set[64] = {};
    if (!set[ctx->device & 63]) {
        CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cap));
        set[ctx->device & 63] = true;
    }
    return launch_pdl(ctx, true, kern, dim3(grid), dim3(NB * 128 + 64), smem, mk, mv, a, stages,
                      q_rows);
}
template <bool BF, int HD>
static int tt_split(cw_ctx* ctx, const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv,
                    int grid) {
    if constexpr (HD <= 128)
        if (a.bm == 256) return tt_go<BF, HD, 2, 1>(ctx, a, mk, mv, grid);
    [[maybe_unused]] const int most = a.max_nodes * a.G;
    if constexpr (HD == 256) {  // at fewer dims short row blocks go to cw_tree_few.cu
        if (most <= 32) return tt_go<BF, HD, 1, 4>(ctx, a, mk, mv, grid);
        if (most <= 64) return tt_go<BF, HD, 1, 2>(ctx, a, mk, mv, grid);
    }
    return tt_go<BF, HD, 1, 1>(ctx, a, mk, mv, grid);
}
template <bool BF>
static int tt_dims(cw_ctx* ctx, const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv,
                   int grid) {
    if (a.D <= 64) return tt_split<BF, 64>(ctx, a, mk, mv, grid);
    if (a.D <= 128) return tt_split<BF, 128>(ctx, a, mk, mv, grid);
    return tt_split<BF, 256>(ctx, a, mk, mv, grid);
}

int tree_tc_launch(cw_ctx* ctx, const TreeArgs& a, uint32_t type, int grid) {
    const bool bf = type == CW_GGUF_BF16;
    CUtensorMap mk, mv;
    CW_TRY(tt_map(&mk, a.k, a, bf));
    CW_TRY(tt_map(&mv, a.v, a, bf));
    if (tt_few_takes(a)) return tt_few_launch(ctx, a, mk, mv, bf, grid);
    return bf ? tt_dims<true>(ctx, a, mk, mv, grid) : tt_dims<false>(ctx, a, mk, mv, grid);
}

}  // namespace cw
