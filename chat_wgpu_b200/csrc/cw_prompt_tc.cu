// cw_prompt_tc.cu -- cw_prompt_attention over 16-bit types on the 5th-generation tensor
// cores (tcgen05, operands staged by TMA, accumulators in TMEM).
//
// Per tile of 128 keys and block of 128 query rows (one TMEM lane a row, row = token * G +
// query head of the kv head):
//
//   S [128 x 128]  = Q K^T   both from shared memory (128-byte swizzled)
//   P [128 x 128]  = 2^(c S - ref), rounded to the type, over the first half of S's columns
//   O [128 x D]   += P V     P from TMEM, V as it lies in memory (keys x dims)
//
// Up to 128 dims two row blocks share a CTA and its K and V tiles: while one block's weights
// are formed the tensor core works on the other's products.  Past 128 dims O fills half of
// TMEM, so there is one row block with two buffers of scores.  A stage of the K/V ring is
// 128 keys of 128 dims at most.
//
// Warps: 4 softmax warps a row block, a thread per row, so row maxima and sums need no
// exchange and no warp waits for another; one warp each to copy, to issue products, to
// find the next item, and to look for values that are not finite.  O is rescaled only when
// a row's maximum has grown by 2^8 since its last reference.  Weights are rounded to the
// type for the second product; the row's sum is taken over the rounded weights, so that a
// constant v comes out exact.
//
// Unseen keys weigh 0, but 0 times a value that is not finite is NaN.  So in the tiles
// that rows see differently (the diagonal, the window's edge) one warp looks V over while
// the weights are formed, and where it finds such values the threads add that tile's
// product themselves, from what each row sees.
#include <algorithm>
#include <mutex>

#include "cw_prompt.cuh"
#include "cw_tree_tc.cuh"

namespace cw {

constexpr int PT_KEYS = 128;    // keys of a tile
constexpr int PT_RING = 2;      // items found ahead
constexpr int PT_LOOKS = 8;     // tiles looked over ahead (the ring holds 5 V tiles at most)
constexpr int PT_STAGES = 10;   // most stages

struct PtItem {
    PromptItem it;
    int head, more;  // more = 0: there are no more items
};

struct PtBars {
    uint64_t full[PT_STAGES], empty[PT_STAGES];
    uint64_t item_full[PT_RING], item_empty[PT_RING];
    uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], pv[2];  // s, p: by buffer of scores
    uint64_t ask[PT_LOOKS], look[PT_LOOKS], done;
    uint32_t tmem, failed, odd[PT_LOOKS], skip[2];
    PtItem item[PT_RING];
};

template <int HD> struct PtShape {
    static constexpr int NB = HD <= 128 ? 2 : 1;             // row blocks
    static constexpr int SB = 3 - NB;                        // buffers of scores of a block
    static constexpr int HALVES = HD <= 128 ? 1 : HD / 128;  // stages of a K or V tile
    static constexpr int COLS = HD / 64 / HALVES;            // 64-dim columns of a stage
    static constexpr int STAGE = COLS * PT_KEYS * 128;
    static constexpr int STAGES = HD == 64 ? 10 : 5;
    static constexpr int QCOL = 128 * 128;                   // bytes of a column of queries
    static constexpr int QBLOCK = HD / 64 * QCOL;
    static constexpr int TCOLS = SB * PT_KEYS + HD;          // TMEM columns of a row block
    static constexpr int THREADS = NB * 128 + 128;
    static constexpr size_t SMEM = (size_t)NB * QBLOCK + STAGES * STAGE + sizeof(PtBars);
    static_assert(SMEM <= 232448, "shared memory of a block");
    static_assert(STAGES <= PT_STAGES && STAGES / 2 + 1 < PT_LOOKS, "rings");
};

// What a row block of an item sees: tiles [lo, hi), and the keys that all of its rows see.
struct PtBlock {
    int lo, hi, all0, all1;
    __device__ __forceinline__ bool in(int i) const { return i >= lo && i < hi; }
    __device__ __forceinline__ bool mixed(int i) const {
        return i * PT_KEYS < all0 || i * PT_KEYS + PT_KEYS - 1 > all1;
    }
};
__device__ __forceinline__ PtBlock pt_block(const PromptArgs& a, const PromptItem& it, int b,
                                            int tpb) {
    PtBlock x = {0, 0, 0, 0};
    const int t0 = b * tpb, t1 = min(t0 + tpb, it.rows);
    if (t0 >= t1) return x;
    const int first = a.window > 0 ? max(0, it.past + t0 - a.window + 1) : 0;
    const int end = min(it.keys, it.past + t1);
    if (end <= first) return x;
    x.lo = first / PT_KEYS;
    x.hi = (end + PT_KEYS - 1) / PT_KEYS;
    x.all0 = a.window > 0 ? it.past + t1 - 1 - a.window + 1 : 0;
    x.all1 = min(it.past + t0, it.keys - 1);
    return x;
}
// The tiles of an item's row blocks together.
template <int NB> struct PtTiles {
    PtBlock b[NB];
    int lo, hi;
    __device__ __forceinline__ PtTiles(const PromptArgs& a, const PromptItem& it, int tpb) {
        lo = 1 << 30;
        hi = 0;
#pragma unroll
        for (int i = 0; i < NB; i++) {
            b[i] = pt_block(a, it, i, tpb);
            if (b[i].hi > b[i].lo) lo = min(lo, b[i].lo), hi = max(hi, b[i].hi);
        }
        lo = min(lo, hi);
    }
    __device__ __forceinline__ bool mixed(int i) const {
        bool x = false;
#pragma unroll
        for (int j = 0; j < NB; j++) x |= b[j].in(i) && b[j].mixed(i);
        return x;
    }
};

__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
        "r"(idesc), "r"(accumulate)
        : "memory");
}
// 64 dims from x of 128 keys of a head.
__device__ __forceinline__ void pt_copy(void* dst, const CUtensorMap* map, int x, int head, int row,
                                        uint64_t* bar) {
    tt_copy_q(dst, map, x, head, row, bar);
}
// 32 bytes at a 32-byte boundary.
__device__ __forceinline__ void pt_store32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// A tile's product by the threads, a row each: O += the weights of the row's P times the
// values that it sees, keys [lo, hi] of the tile.  `first`: there is no O before.
template <bool BF>
__device__ __noinline__ void pt_careful(uint32_t t_p, uint32_t t_o, const uint8_t* const* v, int D,
                                        int lo, int hi, bool first) {
    for (int d0 = 0; d0 < D; d0 += 8) {
        uint32_t o[8];
        tt_ld8(t_o + d0, o);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = first ? 0.f : __uint_as_float(o[e]);
        const uint8_t* col = v[d0 >> 7] + ((d0 >> 6) & 1) * (PT_KEYS * 128);
        const int chunk = (d0 >> 3) & 7;
#pragma unroll 1
        for (int j = 0; j < PT_KEYS; j++) {
            uint32_t p2 = tt_ld1(t_p + (j >> 1));
            asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(p2)::"memory");
            const float p = tt_value<BF>(j & 1 ? p2 >> 16 : p2 & 0xffffu);
            const uint4 w = *(const uint4*)(col + j * 128 + ((chunk ^ (j & 7)) << 4));
            const uint32_t y[4] = {w.x, w.y, w.z, w.w};
            if (j >= lo && j <= hi) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    x[e] = fmaf(p, tt_value<BF>(e & 1 ? y[e >> 1] >> 16 : y[e >> 1] & 0xffffu), x[e]);
            }
            __syncwarp();
        }
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = __float_as_uint(x[e]);
        tt_st<8>(t_o + d0, o);
        tt_wait_st();
    }
}

template <bool BF, int HD>
__global__ void __launch_bounds__(PtShape<HD>::THREADS, 1)
    k_prompt_tc(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PromptArgs a,
                int tpb, int items) {
    typedef PtShape<HD> Z;
    constexpr int NB = Z::NB, SB = Z::SB, HALVES = Z::HALVES, COLS = Z::COLS, STAGE = Z::STAGE;
    constexpr int STAGES = Z::STAGES, TCOLS = Z::TCOLS;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t* s_q = sm;  // [NB][HD / 64][128][128]
    uint8_t* ring = sm + NB * Z::QBLOCK;
    PtBars* bars = (PtBars*)(ring + STAGES * STAGE);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // the swizzle counts from 1024-byte boundaries; no static shared memory precedes
    if (smem_addr(sm) & 1023) {
        if (tid == 0) prompt_bad(a);
        return;
    }
    if (warp == 0) tmem_alloc(&bars->tmem, 512);
    if (tid == 32) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int s = 0; s < PT_RING; s++) {
            mbar_init(&bars->item_full[s], 1);
            mbar_init(&bars->item_empty[s], 3 + NB * 4);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&bars->q_full[b], 1);
            mbar_init(&bars->q_empty[b], 1);
            mbar_init(&bars->s_full[b], 1);
            mbar_init(&bars->p_full[b], 4);
            mbar_init(&bars->pv[b], 1);
            bars->skip[b] = 0;
        }
        for (int i = 0; i < PT_LOOKS; i++) {
            mbar_init(&bars->ask[i], 1);
            mbar_init(&bars->look[i], 1);
        }
        mbar_init(&bars->done, 1);
        bars->failed = 0;
        fence_mbar_init();
    }
    pdl_wait();  // the setup above overlaps the launch before
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem = bars->tmem;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return tt_wait(bar, parity, &bars->failed, a.status);
    };
    auto all = [&](uint64_t* bar, uint32_t parity) {  // the same answer for the warp
        return __all_sync(FULL, wait(bar, parity)) != 0;
    };
    // the item that every role works on, in the same order; false: no more
    int n_item = 0;
    PtItem now;
    auto next = [&]() {
        const int s = n_item % PT_RING;
        if (!all(&bars->item_full[s], n_item / PT_RING)) return false;
        now = bars->item[s];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->item_empty[s]);
        n_item++;
        return now.more != 0;
    };
    constexpr TtTile tile = {1024, PT_KEYS * 128};
    TtPlace at = {0, 0};

    // two row blocks: 168 registers a thread at the start, 208 for the softmax warps of 80
    // left to the others (2 x 128 x 208 + 128 x 80 of 384 x 168)
    if (warp >= NB * 4) {
    if constexpr (NB == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == NB * 4) {  // ---- copies
        int q_count[2] = {0, 0};
        int filled = 0, asks = 0;  // stages filled so far, V tiles to be looked over
        bool ok = true;
        if (tt_elect()) {
            tma_prefetch_desc(&map_q);
            tma_prefetch_desc(&map_k);
            tma_prefetch_desc(&map_v);
        }
        __syncwarp();
        auto load = [&](const CUtensorMap* map, int i) {  // keys of tile i
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                if (h * 128 >= a.D) continue;
                const int s = at.stage;
                if (filled >= STAGES) ok = ok && all(&bars->empty[s], at.phase ^ 1);
                if (ok && tt_elect()) {
                    const int cols = min(COLS, (a.D - h * 128 + 63) / 64);
                    mbar_expect_tx(&bars->full[s], cols * PT_KEYS * 128);
                    for (int c = 0; c < cols; c++)
                        pt_copy(ring + s * STAGE + c * PT_KEYS * 128, map, h * 128 + c * 64, now.head,
                                now.it.key0 + i * PT_KEYS, &bars->full[s]);
                }
                __syncwarp();
                filled += ok;
                if (ok) at.next(STAGES);
            }
        };
        while (ok && next()) {
            const PtTiles<NB> t(a, now.it, tpb);
            if (t.lo >= t.hi) continue;
            load(&map_k, t.lo);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (t.b[b].lo >= t.b[b].hi) continue;
                if (q_count[b] > 0) ok = ok && all(&bars->q_empty[b], q_count[b] - 1);
                if (ok && tt_elect()) {
                    const int cols = (a.D + 63) / 64;
                    mbar_expect_tx(&bars->q_full[b], cols * tpb * a.G * 128);
                    for (int c = 0; c < cols; c++)
                        tt_copy_q(s_q + b * Z::QBLOCK + c * Z::QCOL, &map_q, c * 64, now.head * a.G,
                                  now.it.row0 + b * tpb, &bars->q_full[b]);
                }
                __syncwarp();
                q_count[b] += ok;
            }
            for (int i = t.lo; i < t.hi && ok; i++) {
                if (NB == 1 && i + 1 < t.hi) load(&map_k, i + 1);
                load(&map_v, i);
                if (t.mixed(i)) {
                    if (ok && tt_elect()) mbar_arrive(&bars->ask[asks % PT_LOOKS]);
                    __syncwarp();
                    asks++;
                }
                if (NB == 2 && i + 1 < t.hi) load(&map_k, i + 1);
            }
        }
        if (!ok) {  // copies in flight land before the block may end
            for (int s = 0; s < STAGES; s++)
                if (filled >= STAGES || s < at.stage)
                    (void)mbar_wait(&bars->full[s], s < at.stage ? at.phase : at.phase ^ 1,
                                    TT_WAIT_NS);
            for (int b = 0; b < NB; b++)
                if (q_count[b] > 0) (void)mbar_wait(&bars->q_full[b], (q_count[b] - 1) & 1, TT_WAIT_NS);
        }
    } else if (warp == NB * 4 + 1) {  // ---- products
        constexpr uint32_t id_s = tt_idesc<BF>(PT_KEYS, false, false);
        const uint64_t q0 = umma_desc_sw128(smem_addr(s_q)), kv0 = tt_desc(smem_addr(ring), tile);
        const int steps = (a.D + 15) / 16, halves = HALVES == 1 || a.D <= 128 ? 1 : HALVES;
        int n[2] = {0, 0}, q_count[2] = {0, 0};  // tiles and items of each row block
        bool ok = true;
        while (ok && next()) {
            const PtTiles<NB> t(a, now.it, tpb);
            int done_s[NB];  // tiles of this item whose scores were asked for
#pragma unroll
            for (int b = 0; b < NB; b++) done_s[b] = 0;
            // S = Q K^T of row block b, tile i, whose K is at place k
            auto scores = [&](int b, const TtPlace& k) {
                const int m = n[b] + done_s[b], sb = NB == 2 ? b : m & 1;
                if (done_s[b] == 0) ok = ok && all(&bars->q_full[b], q_count[b]++);
                TtPlace x = k;
#pragma unroll
                for (int h = 0; h < HALVES; h++) {
                    if (h >= halves) continue;
                    ok = ok && all(&bars->full[x.stage], x.phase);
                    tc_fence_after();
                    if (ok && tt_elect()) {
                        const uint32_t d = tmem + b * TCOLS + (NB == 2 ? 0 : sb * PT_KEYS);
                        const uint64_t dk = kv0 + ((x.stage * STAGE) >> 4);
                        const uint64_t dq = q0 + ((b * Z::QBLOCK + h * 2 * Z::QCOL) >> 4);
#pragma unroll
                        for (int s = 0; s < COLS * 4; s++)
                            if (h * 8 + s < steps)
                                umma_f16(d, dq + (((s >> 2) * Z::QCOL + (s & 3) * 32) >> 4),
                                         dk + (((s >> 2) * tile.col + (s & 3) * 32) >> 4), id_s,
                                         h + s > 0);
                    }
                    __syncwarp();
                    x.next(STAGES);
                }
                done_s[b]++;
                if (ok && tt_elect()) {
                    tc_commit(&bars->s_full[sb]);
                    if (done_s[b] == t.b[b].hi - t.b[b].lo) tc_commit(&bars->q_empty[b]);
                }
                __syncwarp();
            };
            // O += P V of row block b, tile i, whose V is at place v
            auto values = [&](int b, int i, const TtPlace& v) {
                const int m = n[b] + i - t.b[b].lo, sb = NB == 2 ? b : m & 1;
                TtPlace x = v;
                for (int h = 0; h < halves; h++, x.next(STAGES))
                    ok = ok && all(&bars->full[x.stage], x.phase);
                ok = ok && all(&bars->p_full[sb], NB == 2 ? m : m >> 1);
                tc_fence_after();
                const bool skip = *(volatile uint32_t*)&bars->skip[sb];
                if (ok && tt_elect()) {
                    const uint32_t p = tmem + b * TCOLS + (NB == 2 ? 0 : sb * PT_KEYS);
                    x = v;
                    for (int h = 0; h < halves && !skip; h++, x.next(STAGES)) {
                        const uint64_t dv = kv0 + ((x.stage * STAGE) >> 4);
                        const uint32_t id_o =
                            tt_idesc<BF>(min(128, (a.D - h * 128 + 15) & ~15), false, true);
#pragma unroll
                        for (int s = 0; s < PT_KEYS / 16; s++)
                            pt_mma_ts(tmem + b * TCOLS + SB * PT_KEYS + h * 128, p + 8 * s,
                                      dv + ((s * 2 * tile.group) >> 4), id_o, s > 0 || i > t.b[b].lo);
                    }
                    tc_commit(&bars->pv[b]);
                }
                __syncwarp();
            };
            auto release = [&](TtPlace& x) {  // a K or V tile, by the products issued so far
                for (int h = 0; h < halves; h++, x.next(STAGES)) {
                    if (ok && tt_elect()) tc_commit(&bars->empty[x.stage]);
                    __syncwarp();
                }
            };
            if (t.lo < t.hi) {
#pragma unroll
                for (int b = 0; b < NB; b++)
                    if (t.b[b].in(t.lo)) scores(b, at);
                release(at);
            }
            for (int i = t.lo; i < t.hi && ok; i++) {
                const bool more = i + 1 < t.hi;
                if (NB == 1) {
                    if (more) {
                        scores(0, at);
                        release(at);
                    }
                    values(0, i, at);
                    release(at);
                } else {
                    TtPlace k = at;  // V of tile i, then K of tile i + 1
                    k.next(STAGES);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        if (t.b[b].in(i)) values(b, i, at);
                        if (b == NB - 1) release(at);
                        if (more && t.b[b].in(i + 1)) scores(b, k);
                    }
                    if (more) release(at);
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b++) n[b] += t.b[b].hi - t.b[b].lo;
        }
        // every product issued has ended before the block frees its TMEM
        if (tt_elect()) {
            tc_commit(&bars->done);
            (void)mbar_wait(&bars->done, 0, TT_WAIT_NS);
        }
        __syncwarp();
    } else if (warp == NB * 4 + 2) {  // ---- which item comes next
        if (blockIdx.x == 0) prompt_check(a, lane, 32);
        int count = 0;
        auto give = [&](const PtItem& x) {
            const int s = count % PT_RING;
            if (count >= PT_RING && !all(&bars->item_empty[s], count / PT_RING - 1)) return false;
            if (lane == 0) {
                bars->item[s] = x;
                mbar_arrive(&bars->item_full[s]);
            }
            __syncwarp();
            count++;
            return true;
        };
        // long items first; every second round of the CTAs goes the other way
        bool ok = true;
        for (int round = 0; ok && round * (int)gridDim.x < items; round++) {
            const int c = round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
            const int x = round * gridDim.x + c;
            if (x >= items) continue;
            PtItem p;
            p.it = prompt_item(a, a.slots - 1 - x / a.K);
            p.head = x % a.K;
            p.more = 1;
            if (p.it.rows > 0) ok = give(p);
        }
        PtItem end = {};
        if (ok) give(end);
    } else {  // ---- values that are not finite, in mixed tiles
        int looks = 0;
        bool ok = true;
        while (ok && next()) {
            const PtTiles<NB> t(a, now.it, tpb);
            const int halves = HALVES == 1 || a.D <= 128 ? 1 : HALVES;
            if (t.lo < t.hi) at.skip(halves, STAGES);
            for (int i = t.lo; i < t.hi && ok; i++) {
                const bool more = i + 1 < t.hi;
                if (NB == 1 && more) at.skip(halves, STAGES);
                if (t.mixed(i)) {
                    uint32_t bits = 0;
                    constexpr uint32_t e = BF ? 0x7f807f80u : 0x7c007c00u;
                    constexpr uint32_t one = BF ? 0x00800080u : 0x04000400u;
                    TtPlace x = at;
                    // asked for once the stage's copy before is over: its phase cannot be
                    // taken for the one before, and the stage is held until P is there
                    ok = all(&bars->ask[looks % PT_LOOKS], looks / PT_LOOKS);
                    for (int h = 0; h < halves && ok; h++, x.next(STAGES)) {
                        ok = all(&bars->full[x.stage], x.phase);
                        const uint8_t* v = ring + x.stage * STAGE;
                        const int n = min(COLS, (a.D - h * 128 + 63) / 64) * PT_KEYS * 128;
#pragma unroll 4
                        for (int o = lane * 16; o < n; o += 512) {
                            const uint4 w = *(const uint4*)(v + o);
                            // all exponent bits set: one more carries into the sign's place
                            bits |= ((w.x & e) + one) | ((w.y & e) + one) | ((w.z & e) + one) |
                                    ((w.w & e) + one);
                        }
                    }
                    const bool odd = __any_sync(FULL, (bits & 0x80008000u) != 0);
                    if (lane == 0) {
                        bars->odd[looks % PT_LOOKS] = odd;
                        mbar_arrive(&bars->look[looks % PT_LOOKS]);
                    }
                    __syncwarp();
                    looks++;
                }
                at.skip(halves, STAGES);
                if (NB == 2 && more) at.skip(halves, STAGES);
            }
        }
    }
    } else {  // ---- softmax: a thread per row
        if constexpr (NB == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int b = warp >> 2, m = tid & 127;
        const uint32_t lanes = tmem + b * TCOLS + ((uint32_t)(warp & 3) << 21);
        const uint32_t t_o = lanes + SB * PT_KEYS;
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
        const int tok = b * tpb + m / a.G, g = m - m / a.G * a.G;  // of the item; query head
        const bool mine = m < tpb * a.G;
        int n = 0, looks = 0;
        bool ok = true;
        while (ok && next()) {
            const PtTiles<NB> t(a, now.it, tpb);
            const PtBlock& blk = t.b[b];
            const bool row = mine && tok < now.it.rows;
            const bool work = __any_sync(FULL, row);
            const int lim = row ? min(now.it.past + tok, now.it.keys - 1) : -1;
            const int low = a.window > 0 ? max(0, now.it.past + tok - a.window + 1) : 0;
            float top = -INFINITY, ref = -INFINITY, sum = 0.f;
            const int halves = HALVES == 1 || a.D <= 128 ? 1 : HALVES;
            TtPlace v = at;  // of tile i's V
            if (t.lo < t.hi) v.skip(halves, STAGES);
            for (int i = t.lo; i < t.hi && ok; i++) {
                const bool more = i + 1 < t.hi, union_mixed = t.mixed(i);
                if (NB == 1 && more) v.skip(halves, STAGES);
                const int look = looks;
                looks += union_mixed;
                const TtPlace vi = v;
                v.skip(halves * (NB == 2 && more ? 2 : 1), STAGES);
                if (!blk.in(i)) continue;
                const int sb = NB == 2 ? b : n & 1, kt = i * PT_KEYS;
                const bool mixed = blk.mixed(i);
                ok = all(&bars->s_full[sb], NB == 2 ? n : n >> 1);
                tc_fence_after();
                const uint32_t t_s = lanes + (NB == 2 ? 0 : sb * PT_KEYS);
                if (work) {
                    float s[PT_KEYS];
#pragma unroll
                    for (int c = 0; c < PT_KEYS; c += 32) tt_ld32(t_s + c, (uint32_t*)s + c);
#pragma unroll
                    for (int c = 0; c < PT_KEYS; c += 32) tt_wait_ld32((uint32_t*)s + c);
                    if (cap) {
#pragma unroll
                        for (int j = 0; j < PT_KEYS; j++) s[j] = capped(s[j]);
                    }
                    if (mixed) {
#pragma unroll
                        for (int j = 0; j < PT_KEYS; j++)
                            if (j < low - kt || j > lim - kt) s[j] = -INFINITY;
                    }
                    float t0 = top, t1 = top, t2 = top, t3 = top;
#pragma unroll
                    for (int j = 0; j < PT_KEYS; j += 4) {
                        t0 = fmaxf(t0, s[j]);
                        t1 = fmaxf(t1, s[j + 1]);
                        t2 = fmaxf(t2, s[j + 2]);
                        t3 = fmaxf(t3, s[j + 3]);
                    }
                    top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
                    const float want = top == -INFINITY ? -INFINITY : top * c2 - TT_LIFT<BF>;
                    if (i == blk.lo) {
                        ref = want;
                    } else if (__any_sync(FULL, row && want - ref > 8.f)) {
                        const float fix = ref == -INFINITY ? 0.f : tt_exp2(ref - want);
                        // O holds the tiles so far (two row blocks: since the scores came)
                        if (NB == 1) ok = ok && all(&bars->pv[b], n - 1);
                        tc_fence_after();
                        sum *= fix;
                        ref = want;
#pragma unroll 1
                        for (int c = 0; c < a.D; c += 16) {
                            uint32_t o[16];
                            tt_load<16>(t_o + c, o);
#pragma unroll
                            for (int j = 0; j < 16; j++)
                                o[j] = __float_as_uint(__uint_as_float(o[j]) * fix);
                            tt_st<16>(t_o + c, o);
                        }
                    }
                    const float from = ref == -INFINITY ? 0.f : ref;
                    float l0 = 0.f, l1 = 0.f;
#pragma unroll
                    for (int c = 0; c < PT_KEYS; c += 64) {
                        uint32_t p[32];
#pragma unroll
                        for (int j = 0; j < 64; j++) s[c + j] = tt_exp2(fmaf(s[c + j], c2, -from));
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            p[j] = tt_pack<BF>(s[c + 2 * j], s[c + 2 * j + 1], l0);
                            p[j + 1] = tt_pack<BF>(s[c + 2 * j + 2], s[c + 2 * j + 3], l1);
                        }
                        tt_st<32>(t_s + c / 2, p);
                    }
                    sum += l0 + l1;
                    tt_wait_st();
                }
                bool odd = false;
                if (mixed) {
                    ok = ok && all(&bars->look[look % PT_LOOKS], look / PT_LOOKS);
                    odd = *(volatile uint32_t*)&bars->odd[look % PT_LOOKS];
                    if (odd && ok && work) {
                        const uint8_t* vt[2];
                        TtPlace x = vi;
                        for (int h = 0; h < halves; h++, x.next(STAGES)) {
                            ok = ok && all(&bars->full[x.stage], x.phase);
                            vt[h] = ring + x.stage * STAGE;
                        }
                        if (i > blk.lo) ok = ok && all(&bars->pv[b], n - 1);
                        tc_fence_after();
                        if (ok)
                            pt_careful<BF>(t_s, t_o, vt, a.D, low - kt, lim - kt, i == blk.lo);
                    }
                }
                if ((warp & 3) == 0 && lane == 0) bars->skip[sb] = odd;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->p_full[sb]);
                n++;
            }
            at = v;
            // ---- the item's end
            const bool none = blk.lo >= blk.hi;
            if (!none) {
                ok = ok && all(&bars->pv[b], n - 1);
                tc_fence_after();
            }
            if (!work || !ok) continue;
            const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
            uint16_t* out = (uint16_t*)a.out +
                            ((long long)(now.it.row0 + tok) * a.H + now.head * a.G + g) * a.D;
            const bool wide = ((uintptr_t)out & 31) == 0 && (a.D & 15) == 0;
#pragma unroll 1
            for (int c = 0; c < a.D; c += 16) {
                uint32_t o[16], w[8];
                __syncwarp();
                if (!none) tt_load<16>(t_o + c, o);
                float unused = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    w[j] = none || inv == 0.f
                               ? 0u
                               : tt_pack<BF>(__uint_as_float(o[2 * j]) * inv,
                                             __uint_as_float(o[2 * j + 1]) * inv, unused);
                if (!row) continue;
                if (wide) {
                    pt_store32(out + c, w);
                } else {
                    *(uint4*)(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                    if (c + 8 < a.D) *(uint4*)(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                }
            }
            __syncwarp();
            tc_fence_before();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

static PFN_cuTensorMapEncodeTiled_v12000 pt_encode_fn() {
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

// Rows of `heads` heads as [rows][heads][D], boxes of 64 dims (zeros past D) by
// `box_heads` heads by `box_rows` rows.
static int pt_map(CUtensorMap* map, const void* base, const PromptArgs& a, bool bf, int heads,
                  int rows, long long stride, int box_heads, int box_rows) {
    auto enc = pt_encode_fn();
    CW_CHECK(enc, CW_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    if (rows == 1) stride = (long long)heads * a.D;  // not used, and may be anything
    cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)heads, (cuuint64_t)rows};
    cuuint64_t strides[2] = {(cuuint64_t)a.D * 2, (cuuint64_t)stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                     const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CW_CHECK(r == CUDA_SUCCESS, CW_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return CW_OK;
}

bool prompt_tc_takes(const PromptArgs& a, uint32_t type) {
    const long long strides = (a.n_rows > 1 ? a.q_stride : 0) |
                              (a.n_keys > 1 ? a.k_stride | a.v_stride : 0);
    return type != CW_GGUF_F32 && a.D % 8 == 0 && a.G <= 128 && a.scale > 0.f && strides % 8 == 0 &&
           (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0;
}

template <bool BF, int HD> static int pt_go(cw_ctx* ctx, PromptArgs& a) {
    typedef PtShape<HD> Z;
    auto kern = k_prompt_tc<BF, HD>;
    const int tpb = 128 / a.G;  // tokens of a row block
    a.bt = Z::NB * tpb;
    a.slots = a.n_rows / a.bt + a.n_req;
    const long long items = (long long)a.slots * a.K;
    CW_CHECK(items < (1ll << 30), CW_ERR_UNSUPPORTED, "cw_prompt_attention: too many rows");
    CUtensorMap mq, mk, mv;
    CW_TRY(pt_map(&mq, a.q, a, BF, a.H, a.n_rows, a.q_stride, a.G, tpb));
    CW_TRY(pt_map(&mk, a.k, a, BF, a.K, a.n_keys, a.k_stride, 1, PT_KEYS));
    CW_TRY(pt_map(&mv, a.v, a, BF, a.K, a.n_keys, a.v_stride, 1, PT_KEYS));
    static bool set[64] = {};
    if (!set[ctx->device & 63]) {
        CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)Z::SMEM));
        set[ctx->device & 63] = true;
    }
    const int grid = (int)std::min<long long>(items, ctx->sm_count);
    CW_TRY(launch_pdl(ctx, true, kern, dim3(grid), dim3(Z::THREADS), Z::SMEM, mq, mk, mv, a, tpb,
                      (int)items));
    return check_launch("prompt_attention");
}
template <bool BF> static int pt_dims(cw_ctx* ctx, PromptArgs& a) {
    if (a.D <= 64) return pt_go<BF, 64>(ctx, a);
    if (a.D <= 128) return pt_go<BF, 128>(ctx, a);
    return pt_go<BF, 256>(ctx, a);
}
int prompt_tc_launch(cw_ctx* ctx, PromptArgs& a, uint32_t type) {
    return type == CW_GGUF_BF16 ? pt_dims<true>(ctx, a) : pt_dims<false>(ctx, a);
}

}  // namespace cw
