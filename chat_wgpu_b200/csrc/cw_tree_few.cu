// cw_tree_few.cu -- cw_tree_attention over 16-bit caches where a request has few query
// rows per kv head (64 at most): decode steps and small trees.
//
// With few rows the products are turned over: keys and head dims, of which there are
// always enough, take the 128-row side of the tensor core, the N (16, 32 or 64) query
// rows its column side.  Per 128-key tile
//
//   S^T [128 keys x N] = K Q^T      K as it lies in memory, Q from shared memory
//   P^T [keys x N]     = 2^(c S^T - ref), rounded to the type, to shared memory
//   O^T [dims x N]    += V^T P^T    V as it lies in memory (128 dims at a time)
//
// so the tensor work is proportional to the rows, a thread (one key of the tile) forms
// N weights instead of padding rows, and K and V are read from shared memory once
// each.  Bound by the cache's bytes in the tiles: 64 KB at D = 128 is 1.5 us of an SM's
// share of the memory bandwidth, against about 0.3 us of products and 0.5 to 1 us of
// weights.  An item's start and end add 2 to 5 us, which deeper rings do not hide: 32
// requests x 16 nodes at 8192 take 142 us where the bytes alone take 108, 256 x 1 of
// 64 dims at 3001 206 us for 149, five of 256 dims with a window 28 us for 11, 250 x 8
// at 400 110 us for 44.  64 rows want more than the 168 registers that 320 threads leave
// (they are charged as 12 warps): 104 bytes a thread are spilled at 128 dims.
//
// No maximum over keys is formed per tile: each row has a reference in shared memory,
// and only when some weight would pass 2^8 (2^15 in f16; always at a row's first tile)
// the maxima over the 128 lanes are reduced, references raised and O^T rescaled.  The
// division by the weights' sum makes the reference drop out.  A thread sums
// its own key's rounded weights, over lanes once at the item's end.
//
// Scores have two TMEM buffers and weights two in shared memory, so the products of
// neighbouring tiles overlap the weights.  Warps: 2 groups of 4 for the weights, half
// the rows each (one group: 180 us for 135, 32 x 16 at 8192 when it was tried); 1 for TMA;
// 1 whose elected lane issues the products.  Keys that not every row sees, v rows past
// the end, keys without a page and values that are not finite are treated as in
// cw_tree_tc.cu.
#include <algorithm>

#include "cw_tree_tc.cuh"

namespace cw {

template <int HD, int N> struct TfShape {
    static constexpr int COLS = HD / 64;
    static constexpr int SK = 128, STAGE = COLS * SK * 128;
    static constexpr int PB = HD <= 128 ? 2 : 1;    // weight buffers (16 KB each)
    static constexpr int OB = HD <= 128 ? 1 : 2;    // 128-dim blocks of O^T
    static constexpr int Q = COLS * N * 128;        // bytes of an item's queries
    static constexpr int QB = HD <= 128 ? 2 : 1;    // their buffers
    static constexpr uint32_t TMEM = 256;           // 2 N of scores, OB N of O^T
    static_assert((2 + OB) * N <= 256, "TMEM");
};

constexpr int TF_STAGES = 12;
constexpr float TF_NONE = 3.402823466e38f;
template <int N> struct TfBars {
    uint64_t full[TF_STAGES], empty[TF_STAGES];
    uint64_t q_full[2], q_empty[2];                      // [item % QB]
    uint64_t s_full[2], p_full[2], pv[2], done;          // [tile % 2]
    uint32_t tmem, failed, keep;
    uint32_t lost;  // some key has no page
    TreeShared run;
    uint64_t sees[2][N];  // [64 keys][row]
    // what is added to a row's scores: -reference, TF_NONE while it has seen nothing above
    // -inf (any such score passes 2^8, and -inf still weighs 0), -inf past the rows
    alignas(16) float neg[N];
    alignas(16) float fix[N];  // a rescale's factors, or at the item's end 1 / sum
    float sums[4][N];          // each warp's
};

template <bool BF> __device__ __forceinline__ uint32_t tf_pack(float x, float y, float& sx,
                                                               float& sy) {
    uint32_t r;
    if (BF) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
        sx += __uint_as_float(r << 16);
        sy += __uint_as_float(r & 0xffff0000u);
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
        const float2 f = __half22float2(*(const __half2*)&r);
        sx += f.x;
        sy += f.y;
    }
    return r;
}
// Barrier and OR: of one group of weight warps (id 1 or 2), or of both (id 3).
__device__ __forceinline__ bool tf_any(bool x, int id) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)x), "r"(id), "r"(id == 3 ? 256 : 128)
        : "memory");
    return r != 0;
}
// C columns of each lane folded over the warp (C at most 32): halving the columns at
// each exchange leaves lane x column x * C / 32.
template <int C, typename F> __device__ __forceinline__ float tf_fold(float (&v)[C], F op) {
    int width = C;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        if (width > 1) {
            width /= 2;
            const bool upper = threadIdx.x & off;
#pragma unroll
            for (int j = 0; j < C / 2; j++) {
                if (j >= width) break;
                const float keep = upper ? v[j + width] : v[j];
                v[j] = op(keep, __shfl_xor_sync(FULL, upper ? v[j] : v[j + width], off));
            }
        } else {
            v[0] = op(v[0], __shfl_xor_sync(FULL, v[0], off));
        }
    }
    return v[0];
}
__device__ __forceinline__ int tf_order(float x) {  // ordered like the float
    const int i = __float_as_int(x);
    return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float tf_float(int i) {
    return __int_as_float(i ^ ((i >> 31) & 0x7fffffff));
}

template <bool BF, int HD, int N>
__global__ void __launch_bounds__(320, 1)
    k_tree_few(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const __grid_constant__ CUtensorMap map_q, const __grid_constant__ TreeArgs a,
               int stages) {
    typedef TfShape<HD, N> Z;
    constexpr int COLS = Z::COLS, SK = Z::SK, STAGE = Z::STAGE, PB = Z::PB, OB = Z::OB;
    constexpr int QB = Z::QB;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t* s_q = sm;                         // [QB][COLS][N][128]
    uint8_t* ring = sm + QB * Z::Q;
    uint8_t* s_p = ring + stages * STAGE;      // [PB][128 keys][64 rows] of weights
    TfBars<N>* bars = (TfBars<N>*)(s_p + PB * 16384);
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
        mbar_init(&bars->done, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars->q_full[i], 1);
            mbar_init(&bars->q_empty[i], 1);
            mbar_init(&bars->s_full[i], 1);
            mbar_init(&bars->p_full[i], 8);
            mbar_init(&bars->pv[i], 1);
        }
        bars->failed = bars->lost = 0;
        fence_mbar_init();
    }
    pdl_wait();  // the setup above overlaps the launch before
    pdl_trigger();
    TreeRun run = tree_run<320>(a, &bars->run);
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
    const TtTile tile =
        tt_wide(a.D) ? TtTile{COLS * 1024, 1024} : TtTile{1024, SK * 128};

    // The tiles of all items run through the products as one sequence t = 0, 1, ..: the
    // scores of tile t + 1 are formed before the values of tile t, so the ring holds
    // K0, then K(t+1), V(t) in turn.
    if (warp == 8) {  // ---- TMA
        TtFeed<COLS, SK> feed(a, ring, bars->full, bars->empty, &bars->lost, stages, tile);
        if (lane == 0) {
            tma_prefetch_desc(&map_k);
            tma_prefetch_desc(&map_v);
            tma_prefetch_desc(&map_q);
        }
        int before = -1;
        bool one_before = false;
        for (uint32_t item = 0; run.left > 0 && ok; item++) {
            it = tree_next(a, run);
            feed.begin(it);
            const int q = item % QB;
            if (item >= QB) ok = all(&bars->q_empty[q], item / QB - 1);
            if (lane == 0 && ok) {
                // [max_nodes][G] rows of 64 dims a copy; rows of later requests come along
                mbar_expect_tx(&bars->q_full[q], COLS * a.max_nodes * a.G * 128);
                for (int c = 0; c < COLS; c++)
                    tt_copy_q(s_q + q * Z::Q + c * N * 128, &map_q, c * 64, it.head * a.G,
                              it.q.row0, &bars->q_full[q]);
            }
            __syncwarp();
            const int tiles = (it.tiles + 1) / 2;
            for (int i = 0; i < tiles && ok; i++) {
                const int now = feed.place(i);
                ok = feed.load(&map_k, now, all);
                if (one_before) ok = ok && feed.load(&map_v, before, all);
                before = now;
                one_before = true;
            }
        }
        if (one_before && ok) ok = feed.load(&map_v, before, all);
        if (!ok) {
            feed.drain();
            for (int q = 0; q < QB; q++)
                for (int ph = 0; ph < 2; ph++) (void)mbar_wait(&bars->q_full[q], ph, 1000000ull);
        }
    } else if (warp == 9) {  // ---- MMA: the warp waits, one lane issues
        constexpr uint32_t id_s = tt_idesc<BF>(N, false, false);
        constexpr uint32_t id_o = tt_idesc<BF>(N, true, true);
        // with 64 dims O^T's lanes 64.. repeat a neighbouring group and are not read
        const TtTile vt = {tile.group, COLS == 1 ? 1024u : tile.col};
        const uint64_t k0 = tt_desc(smem_addr(ring), tile), v0 = tt_desc(smem_addr(ring), vt),
                       q0 = umma_desc_sw128(smem_addr(s_q)),
                       p0 = tt_desc(smem_addr(s_p), TtTile{1024, 1024});
        const int steps = (a.D + 15) / 16;
        const bool one = tt_elect();
        TtPlace at = {0, 0};
        // O^T (+)= V^T P^T of tile t; the first of an item starts O^T anew
        auto values = [&](uint32_t t, bool first) {
            const int s = at.stage;
            ok = ok && all(&bars->full[s], at.phase);
            at.next(stages);
            ok = ok && all(&bars->p_full[t & 1], t >> 1);
            tc_fence_after();
            if (one && ok) {
                const uint32_t add = first ? *(volatile uint32_t*)&bars->keep : 1u;
                const uint64_t dv = v0 + ((s * STAGE) >> 4),
                               dp = p0 + (((t % PB) * 16384) >> 4);
#pragma unroll
                for (int ob = 0; ob < OB; ob++)
#pragma unroll
                    for (int x = 0; x < SK / 16; x++)
                        umma_f16(tmem + (2 + ob) * N,
                                 dv + ((ob * 2 * tile.col + x * 2 * tile.group) >> 4),
                                 dp + ((x * 2048) >> 4), id_o, x > 0 ? 1u : add);
                tc_commit(&bars->pv[t & 1]);
                tc_commit(&bars->empty[s]);
            }
            __syncwarp();
        };
        uint32_t t = 0;
        bool first = false;
        for (uint32_t item = 0; run.left > 0 && ok; item++) {
            it = tree_next(a, run);
            const int tiles = (it.tiles + 1) / 2, q = item % QB;
            ok = all(&bars->q_full[q], item / QB);
            for (int i = 0; i < tiles && ok; i++, t++) {
                // S^T of tile t.  Its buffer's scores, of tile t - 2, were read before
                // that tile's weights arrived.
                const int s = at.stage;
                ok = ok && all(&bars->full[s], at.phase);
                at.next(stages);
                tc_fence_after();
                if (one && ok) {
                    const uint64_t dk = k0 + ((s * STAGE) >> 4), dq = q0 + ((q * Z::Q) >> 4);
#pragma unroll
                    for (int x = 0; x < HD / 16; x++)
                        if (x < steps)
                            umma_f16(tmem + (t & 1) * N,
                                     dk + (((x >> 2) * tile.col + (x & 3) * 32) >> 4),
                                     dq + (((x >> 2) * N * 128 + (x & 3) * 32) >> 4), id_s,
                                     x > 0);
                    tc_commit(&bars->s_full[t & 1]);
                    tc_commit(&bars->empty[s]);
                    if (i + 1 == tiles) tc_commit(&bars->q_empty[q]);
                }
                __syncwarp();
                if (t > 0) values(t - 1, first);
                first = i == 0;
            }
        }
        if (t > 0 && ok) values(t - 1, first);
        // every product issued has ended before the block frees its TMEM
        if (one) tc_commit(&bars->done);
        (void)mbar_wait(&bars->done, 0, TT_WAIT_NS);
        __syncwarp();
    } else {
        // ---- weights: two groups of 4 warps, half the rows each (C columns from c0).
        // Thread m of a group has key m of the tile, and at the item's end dim m.
        constexpr int C = N / 2;
        const int group = warp >> 2, c0 = group * C, id = 1 + group;
        const int m = tid & 127, half = m >> 6;
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21) + c0, t_o = lanes + 2 * N;
        const float log2e = 1.44269504088896341f;
        const bool cap = a.softcap > 0.f;
        const float c2 = cap ? log2e : a.scale * log2e;
        const float y2 = cap ? 2.f * log2e * a.scale / a.softcap : 0.f;
        float* neg = bars->neg + c0;
        float* fix = bars->fix + c0;
        uint32_t n = 0;
        TtPlace at_v = {0, 0};  // of this tile's V: V0 is the third, or the second and last
        at_v.skip(1, stages);
        while (run.left > 0) {
            it = tree_next(a, run);
            any = true;
            const int tiles = (it.tiles + 1) / 2, rows = it.rows;
            const int key0 = (it.q.tile0 + it.tile) * TR_TILE;
            const int end = min(it.q.keys, key0 + it.tiles * TR_TILE);  // of this piece's keys
            int edge = 0;  // the largest of the item's rows
            if (a.window > 0) {
                for (int node = lane; node < it.q.n; node += 32)
                    edge = max(edge, tree_edge(a, it.q, node * a.G));
                edge = __reduce_max_sync(FULL, edge);
            }
            if (m < C) {
                neg[m] = c0 + m < rows ? TF_NONE : -INFINITY;
                fix[m] = __int_as_float(tf_order(-INFINITY));
            }
            if (tid == 0) bars->keep = 0;
            (void)tf_any(false, id);
            float l[C];
#pragma unroll
            for (int c = 0; c < C; c++) l[c] = 0.f;
            for (int i = 0; i < tiles; i++, n++) {
                const int kt = key0 + i * SK;
                const bool mixed = kt + SK > end || kt + SK > it.q.len || kt < edge;
                at_v.skip(run.left <= 0 && i + 1 == tiles ? 0 : 1, stages);
                if (mixed) {
                    (void)tf_any(false, 3);  // the last tile's sets have been read
                    const int r = tid & 63, h = tid >> 6, k = kt + h * 64;
                    if (r < N && h < 2)
                        bars->sees[h][r] = r < rows && k < end ? tree_sees(a, it.q, r, k) : 0;
                    (void)tf_any(false, 3);
                }
                const uint64_t* sees = bars->sees[half] + c0;
                wait(&bars->s_full[n & 1], n >> 1);
                __syncwarp();
                tc_fence_after();
                // set before the tile's keys were, if one of them has no page
                const bool lost = *(volatile uint32_t*)&bars->lost;
                float s[C];
                // pass 1: the weights' exponents; were some to pass 8, or 15 in f16 (0, and
                // at once at an item's first tile): new references; 2: the exponents again
#pragma unroll 1
                for (int pass = i == 0 ? 0 : 1;;) {
                    tt_load<C>(lanes + (n & 1) * N, (uint32_t*)s);
                    if (cap) {
                        // tanh(y) = 1 - 2 / (1 + e^2y): off by 2^-22, times softcap far
                        // below one rounding of the weight
#pragma unroll
                        for (int c = 0; c < C; c++) {
                            const float y = s[c] * y2;
                            s[c] = a.softcap - __fdividef(2.f * a.softcap,
                                                          1.f + tt_exp2(y > 120.f ? 120.f : y));
                        }
                    }
                    if (mixed) {
#pragma unroll
                        for (int c = 0; c < C; c++)
                            if (!(sees[c] >> (m & 63) & 1)) s[c] = -INFINITY;
                    }
                    if (lost && kt + m < end && !tree_has(a, it.r, kt + m)) {
#pragma unroll
                        for (int c = 0; c < C; c++) s[c] = -INFINITY;
                    }
                    if (pass == 0) {
                        // maxima over the 128 keys: in fix, as ordered whole numbers
#pragma unroll
                        for (int c = 0; c < C; c++) s[c] *= c2;
                        const float top = tf_fold<C>(s, [](float x, float y) { return fmaxf(x, y); });
                        if (lane % (32 / C) == 0)
                            atomicMax((int*)fix + lane * C / 32, tf_order(top));
                        (void)tf_any(false, id);
                        if (m < C) {
                            const float was = -neg[m];
                            const float now =
                                fmaxf(tf_float(__float_as_int(fix[m])) - TT_LIFT<BF>, was);
                            fix[m] = tt_exp2(was - now);
                            if (c0 + m < rows) neg[m] = -now;
                        }
                        (void)tf_any(false, id);
#pragma unroll
                        for (int c = 0; c < C; c++) l[c] *= fix[c];
                        if (i > 0) {
                            wait(&bars->pv[(n - 1) & 1], (n - 1) >> 1);  // O^T: the tiles so far
                            __syncwarp();
                            tc_fence_after();
#pragma unroll 1
                            for (int ob = 0; ob < OB; ob++) {
                                float o[C];
                                tt_load<C>(t_o + ob * N, (uint32_t*)o);
#pragma unroll
                                for (int c = 0; c < C; c++) o[c] *= fix[c];
                                tt_st<C>(t_o + ob * N, (const uint32_t*)o);
                            }
                            tt_wait_st();
                        }
                        (void)tf_any(false, id);  // the factors have been read
                        if (m < C) fix[m] = __int_as_float(tf_order(-INFINITY));
                        pass = 2;
                        continue;
                    }
                    float most = -INFINITY;
#pragma unroll
                    for (int c = 0; c < C; c += 4) {
                        const float4 f = *(const float4*)&neg[c];
                        s[c] = fmaf(s[c], c2, f.x);
                        s[c + 1] = fmaf(s[c + 1], c2, f.y);
                        s[c + 2] = fmaf(s[c + 2], c2, f.z);
                        s[c + 3] = fmaf(s[c + 3], c2, f.w);
                        most = fmaxf(most, fmaxf(fmaxf(s[c], s[c + 1]), fmaxf(s[c + 2], s[c + 3])));
                    }
                    if (pass == 2 || !tf_any(most > 8.f + TT_LIFT<BF>, id)) break;
                    pass = 0;
                }
                // The product that read this weight buffer: with two, that of tile n - 2,
                // which was issued before this tile's scores and so ended before them.
                if (PB == 1 && i > 0) {
                    wait(&bars->pv[(n - 1) & 1], (n - 1) >> 1);
                    __syncwarp();
                }
                uint8_t* p = s_p + (n % PB) * 16384;
#pragma unroll
                for (int c = 0; c < C; c++) s[c] = tt_exp2(s[c]);
#pragma unroll
                for (int c = 0; c < C; c += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        w[e] = tf_pack<BF>(s[c + 2 * e], s[c + 2 * e + 1], l[c + 2 * e],
                                           l[c + 2 * e + 1]);
                    *(uint4*)(p + m * 128 + ((((c0 + c) >> 3) ^ (m & 7)) << 4)) =
                        make_uint4(w[0], w[1], w[2], w[3]);
                }
                if (mixed) {  // v rows past the end, and values that are not finite
                    wait(&bars->full[at_v.stage], at_v.phase);
                    __syncwarp();
                    uint8_t* v = ring + at_v.stage * STAGE;
                    const int live = min(end - kt, SK);
                    bool odd = false;
                    for (int x = tid; x < COLS * SK * 8; x += 256) {
                        const int j = x / (COLS * 8);
                        uint4* w = (uint4*)(v + tile.at(j, x % (COLS * 8)));
                        if (j >= live) *w = make_uint4(0, 0, 0, 0);
                        else odd |= tt_odd8<BF>(*w);
                    }
                    if (tf_any(odd, 3)) {
                        if (i > 0) {
                            wait(&bars->pv[(n - 1) & 1], (n - 1) >> 1);
                        } else {  // O^T starts here: from zeros, kept by the first product
                            uint32_t z[C];
#pragma unroll
                            for (int e = 0; e < C; e++) z[e] = 0;
#pragma unroll 1
                            for (int ob = 0; ob < OB; ob++) tt_st<C>(t_o + ob * N, z);
                            tt_wait_st();
                            if (tid == 0) bars->keep = 1;
                        }
                        __syncwarp();
                        tc_fence_after();
#pragma unroll 1
                        for (int x = 0; x < OB * live; x++) {
                            const int j = x % live, ob = x / live, d = ob * 128 + m;
                            const uint32_t bits =
                                d < HD ? *(const uint16_t*)(v + tile.at(j, d >> 3) + (d & 7) * 2)
                                       : 0u;
                            const bool mine = tt_odd<BF>(bits);
                            if (!__any_sync(FULL, mine)) continue;
                            float o[C];
                            tt_load<C>(t_o + ob * N, (uint32_t*)o);
#pragma unroll
                            for (int e = 0; e < C; e++) {
                                const int c = c0 + e;
                                const uint32_t w = *(const uint16_t*)(
                                    p + j * 128 + (((c >> 3) ^ (j & 7)) << 4) + (c & 7) * 2);
                                if (mine && (bars->sees[j >> 6][c] >> (j & 63) & 1))
                                    o[e] = fmaf(tt_value<BF>(w), tt_value<BF>(bits), o[e]);
                            }
                            __syncwarp();
                            tt_st<C>(t_o + ob * N, (const uint32_t*)o);
                            tt_wait_st();
                        }
                        (void)tf_any(false, 3);  // all have read them
                        for (int x = tid; x < COLS * SK * 8; x += 256) {
                            uint16_t* w = (uint16_t*)(v + tile.at(x / (COLS * 8), x % (COLS * 8)));
                            for (int e = 0; e < 8; e++)
                                if (tt_odd<BF>(w[e])) w[e] = 0;
                        }
                    }
                }
                tt_fence_async();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->p_full[n & 1]);
                at_v.skip(1, stages);
            }
            // ---- the item's end
            const float sum = tf_fold<C>(l, [](float x, float y) { return x + y; });
            if (lane % (32 / C) == 0) bars->sums[warp & 3][c0 + lane * C / 32] = sum;
            wait(&bars->pv[(n - 1) & 1], (n - 1) >> 1);
            (void)tf_any(false, id);
            tc_fence_after();
            const size_t piece = ((size_t)blockIdx.x * 2 + tree_slot(run, it)) * a.bm;
            if (m < C) {
                const int c = c0 + m;
                const float l4 = (bars->sums[0][c] + bars->sums[1][c]) +
                                 (bars->sums[2][c] + bars->sums[3][c]);
                if (c < rows && !it.whole) a.ml[piece + c] = make_float2(-neg[m], l4);
                fix[m] = l4 > 0.f || l4 != l4 ? 1.f / l4 : 0.f;
            }
            (void)tf_any(false, id);
            const int mine = min(max(rows - c0, 0), C);  // this group's rows
#pragma unroll 1
            for (int ob = 0; ob < OB && mine > 0; ob++) {
                const int d = ob * 128 + m;
                float o[C];
                __syncwarp();
                tt_load<C>(t_o + ob * N, (uint32_t*)o);
                if (d >= a.D) continue;
                if (it.whole) {
                    int gi = c0 % a.G;
                    uint16_t* to = (uint16_t*)a.out +
                                   ((long long)(it.q.row0 + c0 / a.G) * a.H + it.head * a.G + gi) *
                                       a.D + d;
                    const long long jump = (long long)(a.H - a.G) * a.D;
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        if (c >= mine) break;
                        const float inv = fix[c], y = inv == 0.f ? 0.f : o[c] * inv;
                        if (BF) *(__nv_bfloat16*)to = __float2bfloat16_rn(y);
                        else *(__half*)to = __float2half_rn(y);
                        to += a.D;  // next head of the group, or the next node's first
                        if (++gi == a.G) {
                            gi = 0;
                            to += jump;
                        }
                    }
                } else {
                    float* to = a.part + (piece + c0) * a.dp + d;
#pragma unroll
                    for (int c = 0; c < C; c++, to += a.dp)
                        if (c < mine) *to = o[c];
                }
            }
            __syncwarp();
            tc_fence_before();
            (void)tf_any(false, id);  // the references are read no more
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

// 64 rows, or 32 of 256 dims (the ring needs three tiles beside the queries); a tile's
// copies have to fit one warp's lanes.
bool tt_few_takes(const TreeArgs& a) {
    const int cols = tt_wide(a.D) || a.D <= 64 ? 1 : a.D <= 128 ? 2 : 4;
    return a.max_nodes * a.G <= (a.D <= 128 ? 64 : 32) && 128 / std::min(a.page, 64) * cols <= 32;
}

template <bool BF, int HD, int N>
static int tf_go(cw_ctx* ctx, const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv,
                 int grid) {
    typedef TfShape<HD, N> Z;
    auto kern = k_tree_few<BF, HD, N>;
    const size_t cap = 232448, fixed = Z::QB * Z::Q + Z::PB * 16384 + sizeof(TfBars<N>);
    const int stages = (int)std::min<size_t>((cap - fixed) / Z::STAGE, TF_STAGES);
    static_assert((cap - fixed) / Z::STAGE >= 3, "K(i+1), V(i) and one in flight");
    static bool set[64] = {};
    if (!set[ctx->device & 63]) {
        CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cap));
        set[ctx->device & 63] = true;
    }
    CUtensorMap mq;
    CW_TRY(tt_map_q(&mq, a, BF));
    return launch_pdl(ctx, true, kern, dim3(grid), dim3(320), fixed + stages * Z::STAGE, mk, mv,
                      mq, a, stages);
}
template <bool BF, int HD>
static int tf_rows(cw_ctx* ctx, const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv,
                   int grid) {
    if (a.bm == 16) return tf_go<BF, HD, 16>(ctx, a, mk, mv, grid);
    if constexpr (HD <= 128)
        if (a.bm == 64) return tf_go<BF, HD, 64>(ctx, a, mk, mv, grid);
    return tf_go<BF, HD, 32>(ctx, a, mk, mv, grid);
}
template <bool BF>
static int tf_dims(cw_ctx* ctx, const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv,
                   int grid) {
    if (a.D <= 64) return tf_rows<BF, 64>(ctx, a, mk, mv, grid);
    if (a.D <= 128) return tf_rows<BF, 128>(ctx, a, mk, mv, grid);
    return tf_rows<BF, 256>(ctx, a, mk, mv, grid);
}
int tt_few_launch(cw_ctx* ctx, const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv,
                  bool bf, int grid) {
    return bf ? tf_dims<true>(ctx, a, mk, mv, grid) : tf_dims<false>(ctx, a, mk, mv, grid);
}

}  // namespace cw
