// cw_prompt_tc.cu -- cw_prompt_attention on the 5th-generation tensor cores (tcgen05,
// operands staged by TMA, accumulators in TMEM): 16-bit types, and f32 as pairs of f16.
//
// Per tile of 128 keys and block of 128 query rows (one TMEM lane a row, row = token * G +
// query head of the kv head):
//
//   S [128 x 128]  = Q K^T   both from shared memory (128-byte swizzled)
//   P [128 x 128]  = 2^(c S - ref), rounded to the type, over half of S's columns
//   O [128 x D]   += P V     P from TMEM, V as it lies in memory (keys x dims)
//
// Up to 128 dims two row blocks share a CTA and its K and V tiles: while one block's weights
// are formed the tensor core works on the other's products.  Past 128 dims O fills half of
// TMEM, so there is one row block with two buffers of scores.  A stage of the K/V ring is
// 128 keys of 128 dims at most.
//
// Warps: 8 softmax warps a row block, two threads to a row with 64 keys of a tile each, which
// tell each other their maxima (a thread to a row kept 128 scores, and its one warp per
// scheduler waited for itself: 16384 bf16 tokens of 32/8 heads 1.88 ms against 1.82); one
// warp each to copy, to issue products (one lane: 1.87 ms without any softmax when the warp
// went together, 1.40 ms alone), to find the next item, and to look for values that are not
// finite.  O is rescaled only when a row's weights have grown by 2^8 (pairs: 2^2) since its last
// reference.
// Weights are rounded to the type for the second product, half a step each at most; the
// row's sum takes them unrounded, which saves two instructions a key.
//
// What bounds it: at 16384 bf16 tokens the products alone, with no softmax between them, take
// 1.40 ms (1570 TFLOP/s, 0.94 of the measured burst peak), all of it 1.8 to 1.9 ms in short
// runs and 2.1 to 2.2 ms in long ones, where the power limit lowers the clock.  The tensor pipe is
// active 55 to 60 % of the time, the special-function unit half of it; the rest is the chain
// scores -> weights -> product of each row block.  Powers of two by polynomials on the FMA
// pipe made it slower in every share tried (1/8 of them: 1.83 -> 1.88 ms; 3/8: 2.00 ms), as
// did leaving out the masked end of the last tile (1.90 -> 1.96 ms): the chain and the power
// count instructions, not one unit's time.
//
// f32 (head_dim <= 128): x 2^s = h + l, s by request and kv head (k, v) or by row and head
// (q), and each product is h h + h l + l h, with l held 2^11 times as large and the sum of the
// small products divided by that when h h begins (a small element's l would sink into f16's
// subnormals: 2^-9 of an element 2^-30 of the largest was lost, and 2^-20 is now; no time
// was).  The tensor cores cut their f32 sums at each step
// by what they have grown to, so the small products come first and a tile's sums are added
// to the row's by the threads (error against 64 bits at 4096 keys 7.1e-6 without either,
// 6.8e-7 with both; a plain f32 form has 1.2e-6).  Bound by shared memory and the tensor
// pipe: 128 rows take 416 KB of operands a tile through it, 3300 cycles at 128 bytes, for
// 3100 cycles of products.  What does not fit pairs (infinities, NaN, magnitudes from 2^60 or
// below 2^-86, rows of very different sizes) is left to the f32 kernel, by request and kv head.
//
// Unseen keys weigh 0, but 0 times a value that is not finite is NaN.  So in the tiles
// that rows see differently (the diagonal, the window's edge) one warp looks V over while
// the weights are formed, and where it finds such values the threads add that tile's
// product themselves, from what each row sees.
//
// Many items are dealt whole, long ones first, rounds of the CTAs going forth and back.  Few
// items over many keys are cut into equal runs of tiles, and a second launch joins them.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "cw_prompt.cuh"
#include "cw_tree_tc.cuh"

namespace cw {

constexpr int PT_KEYS = 128;    // keys of a tile
constexpr int PT_RING = 3;      // items found ahead
constexpr int PT_LOOKS = 8;     // tiles looked over ahead (the ring holds 5 V tiles at most)
constexpr int PT_STAGES = 10;   // most stages
constexpr int PT_PAD = 2;       // tiles that an item's start and end count as
constexpr int PT_CUT = 6;       // items of fewer tiles are not cut
constexpr int PT_LEAST = 4;     // units of a CTA's run where items are cut

// What a row block of an item sees: tiles [lo, hi), all rows the same in [all0, all1).
struct PtBlock {
    int lo, hi, all0, all1;
    __device__ __forceinline__ bool in(int i) const { return i >= lo && i < hi; }
    __device__ __forceinline__ bool mixed(int i) const { return i < all0 || i >= all1; }
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
    const int late = a.window > 0 ? max(0, it.past + t1 - a.window) : 0;  // the last row's first key
    x.all0 = (late + PT_KEYS - 1) / PT_KEYS;
    x.all1 = max(0, min(it.past + t0 + 1, it.keys)) / PT_KEYS;  // up to the first row's last key
    return x;
}
// The tiles of an item's row blocks together, [lo, hi), K and V in the order of the ring: K
// of tile lo, then V of each tile behind K of its own (two row blocks) or of the next one.
// Tiles outside [all0, all1), which may be mixed for a block, are looked over.
template <int NB> struct PtTiles {
    PtBlock b[NB];
    int lo, hi, all0, all1;
    __device__ __forceinline__ void set(const PromptArgs& a, const PromptItem& it, int tpb) {
        lo = all1 = 1 << 30;
        hi = all0 = 0;
#pragma unroll
        for (int i = 0; i < NB; i++) {
            b[i] = pt_block(a, it, i, tpb);
            if (b[i].hi <= b[i].lo) continue;
            lo = min(lo, b[i].lo);
            hi = max(hi, b[i].hi);
            all0 = max(all0, b[i].all0);
            all1 = min(all1, b[i].all1);
        }
        lo = min(lo, hi);
        all0 = min(max(all0, lo), hi);
        all1 = min(max(all1, all0), hi);
    }
    // tiles [x, y) of them only
    __device__ __forceinline__ void clip(int x, int y) {
        lo = max(lo, x);
        hi = max(lo, min(hi, y));
#pragma unroll
        for (int i = 0; i < NB; i++) {
            b[i].lo = max(b[i].lo, x);
            b[i].hi = max(b[i].lo, min(b[i].hi, y));
        }
        all0 = min(max(all0, lo), hi);
        all1 = min(max(all1, all0), hi);
    }
    __device__ __forceinline__ bool look(int i) const { return i < all0 || i >= all1; }
    // tiles looked over before tile i; K and V tiles in the ring before V of tile i
    __device__ __forceinline__ int looks(int i) const { return min(i, all0) - lo + max(0, i - all1); }
    __device__ __forceinline__ int before(int i) const {
        return 2 * (i - lo) + 1 + (NB == 1 && i + 1 < hi);
    }
};
// What every role reads of an item.  more = 0: there are no more items.
template <int NB> struct PtItem {
    PromptItem it;
    int head, more;
    int whole, slot;       // all of its tiles; else where its partial state goes
    float k_back, v_back;  // pairs: what k and v were divided by
    PtTiles<NB> t;
};
// A CTA's run of the units of all items, in slot, kv head, tile order: it begins `off` units
// behind the start of slot's first kv head and has `left`.
struct PtRun {
    long long w[24], off;
    int slot;
};
template <int NB> struct PtBars {
    uint64_t full[PT_STAGES], empty[PT_STAGES];
    uint64_t item_full[PT_RING], item_empty[PT_RING];
    uint64_t q_full[2], q_empty[2], s_full[2], p_half[2], p_full[2], pv[2];  // s, p: by buffer of scores
    uint64_t ask[PT_LOOKS], look[PT_LOOKS], done;
    uint32_t tmem, failed, odd[PT_LOOKS], skip[2];
    float meet[2][2][128];  // what the two threads of a row tell each other
    PtRun run;
    PtItem<NB> item[PT_RING];
};

// HD: head_dim rounded up to 64, 128 or 256.  PAIR: f32 operands as pairs of f16 (HD <= 128),
// whose high and low parts are the two halves of a tile.
template <int HD, bool PAIR> struct PtShape {
    static constexpr int NB = HD <= 128 && !PAIR ? 2 : 1;    // row blocks
    static constexpr int SB = 3 - NB;                        // buffers of scores of a block
    static constexpr int HALVES = PAIR ? 2 : HD <= 128 ? 1 : HD / 128;  // stages of a K or V tile
    static constexpr int WIDTH = PAIR ? HD : 128;            // dims from half to half in memory
    static constexpr int COLS = PAIR ? HD / 64 : HD / 64 / HALVES;      // 64-dim columns of a stage
    static constexpr int STAGE = COLS * PT_KEYS * 128;
    static constexpr int STAGES = HD == 64 ? 10 : 5;
    static constexpr int QCOL = 128 * 128;                   // bytes of a column of queries
    static constexpr int QBLOCK = HALVES * COLS * QCOL;
    static constexpr int OB = PAIR ? 2 : 1;                  // buffers of sums
    static constexpr int TCOLS = SB * PT_KEYS + OB * HD;     // TMEM columns of a row block
    static constexpr int WARPS = NB * 8;                     // softmax warps
    static constexpr int THREADS = WARPS * 32 + 128;
    static constexpr size_t SMEM = (size_t)NB * QBLOCK + STAGES * STAGE + sizeof(PtBars<NB>);
    static_assert(SMEM <= 232448, "shared memory of a block");
    static_assert(STAGES <= PT_STAGES && STAGES / 2 + 1 < PT_LOOKS, "rings");
};
// The place in the ring after n stages.
template <int STAGES> __device__ __forceinline__ TtPlace pt_place(uint32_t n) {
    return {(int)(n % STAGES), n / STAGES & 1};
}

__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
        "r"(idesc), "r"(accumulate)
        : "memory");
}
// The same products with what the accumulator held before divided by 2^PT_LOW first.
constexpr int PT_LOW = 11;
__device__ __forceinline__ void pt_mma_ss_low(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, %4;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "r"(idesc), "n"(PT_LOW)
        : "memory");
}
__device__ __forceinline__ void pt_mma_ts_low(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, %4;\n\t}" ::"r"(d), "r"(a), "l"(b),
        "r"(idesc), "n"(PT_LOW)
        : "memory");
}
// 32 bytes at a 32-byte boundary.
__device__ __forceinline__ void pt_store32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// A wait that was not over at once: bounded, like tt_wait, but out of line and without a look
// at the clock before many tries, which would delay the wake-up.
__device__ __noinline__ bool pt_wait_on(uint64_t* bar, uint32_t parity, uint32_t* failed,
                                        int* status) {
    for (int i = 0; i < 256; i++)
        if (mbar_try_wait(bar, parity)) return true;
    return tt_wait(bar, parity, failed, status);
}
__device__ __forceinline__ bool pt_wait(uint64_t* bar, uint32_t parity, uint32_t* failed,
                                        int* status) {
    return mbar_try_wait(bar, parity & 1) || pt_wait_on(bar, parity & 1, failed, status);
}
// The largest of three, NaN if one is.
__device__ __forceinline__ float pt_max3(float x, float y, float z) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
// Two weights rounded and packed, first in the low half.
template <bool BF> __device__ __forceinline__ uint32_t pt_pack(float x, float y) {
    uint32_t r;
    if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}

// The scores of a row's half of a tile in TMEM, capped, to f32's accuracy.  y: scale / softcap.
__device__ __noinline__ void pt_cap_f32(uint32_t t_s, float softcap, float y) {
#pragma unroll 1
    for (int c = 0; c < PT_KEYS / 2; c += 16) {
        float s[16];
        tt_load<16>(t_s + c, (uint32_t*)s);
#pragma unroll
        for (int j = 0; j < 16; j++) s[j] = softcap * tanhf(s[j] * y);
        tt_st<16>(t_s + c, (uint32_t*)s);
    }
    tt_wait_st();
}
// The same for weights in 16 bits: tanh(y) = 1 - 2 / (1 + e^2y), off by 2^-22, which times a
// softcap of PT_CAP_FAST at most is 2^-14, an eighth of the rounding of an f16 weight.  (Larger
// caps would lose the score in the difference: scores of 8 are off by 0.1 at 1e6.  They are
// told here and not where it is called: two calls there made every kernel of 16-bit types
// 3.5 % slower.)  y2: 2 log2(e) scale / softcap.
constexpr float PT_CAP_FAST = 256.f;
__device__ __noinline__ void pt_cap(uint32_t t_s, float softcap, float y2) {
    if (softcap > PT_CAP_FAST) {
        pt_cap_f32(t_s, softcap, y2 * 0.346573590279972655f);  // ln(2) / 2
        return;
    }
#pragma unroll 1
    for (int c = 0; c < PT_KEYS / 2; c += 32) {
        float s[32];
        tt_load<32>(t_s + c, (uint32_t*)s);
#pragma unroll
        for (int j = 0; j < 32; j++) {
            const float y = s[j] * y2;
            s[j] = softcap - __fdividef(2.f * softcap, 1.f + tt_exp2(y > 120.f ? 120.f : y));
        }
        tt_st32(t_s + c, (uint32_t*)s);
    }
    tt_wait_st();
}
// -inf for the keys of the half outside [lo, hi].
__device__ __noinline__ void pt_hide(uint32_t t_s, int lo, int hi) {
#pragma unroll 1
    for (int c = 0; c < PT_KEYS / 2; c += 32, lo -= 32, hi -= 32) {
        float s[32];
        tt_load<32>(t_s + c, (uint32_t*)s);
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (j < lo || j > hi) s[j] = -INFINITY;
        tt_st32(t_s + c, (uint32_t*)s);
    }
    tt_wait_st();
}

// A tile's product by the threads, two to a row with every other 8 dims each: O += the
// weights of the row's P times the values that it sees, keys [lo, hi] of the tile.  `first`:
// there is no O before.
template <bool BF>
__device__ __noinline__ void pt_careful(uint32_t t_p, uint32_t t_o, const uint8_t* const* v, int D,
                                        int half, int lo, int hi, bool first) {
    for (int d0 = half * 8; d0 < D; d0 += 16) {
        uint32_t o[8];
        tt_ld8(t_o + d0, o);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = first ? 0.f : __uint_as_float(o[e]);
        const uint8_t* col = v[d0 >> 7] + ((d0 >> 6) & 1) * (PT_KEYS * 128);
        const int chunk = (d0 >> 3) & 7;
#pragma unroll 1
        for (int j = 0; j < PT_KEYS; j++) {
            uint32_t p2 = tt_ld1(t_p + (j >> 6) * (PT_KEYS / 2) + ((j & 63) >> 1));
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

// Units of slot s for one kv head: its tiles, and PT_PAD for its start and end.
template <int NB> __device__ int pt_units(const PromptArgs& a, int s, int tpb) {
    const PromptItem it = prompt_item(a, s);
    if (it.rows <= 0) return 0;
    PtTiles<NB> t;
    t.set(a, it, tpb);
    return t.hi - t.lo + PT_PAD;
}
// All threads (NT of them): this CTA's run.  The units of all slots are summed by every CTA,
// a slot to a thread.
template <int NB, int NT>
__device__ void pt_run(const PromptArgs& a, int tpb, PtRun* run, long long& per, long long& left) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // sums of the threads' values before each, and of all
    auto scan = [&](long long mine, long long& total) {
        long long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(FULL, incl, o);
            if (lane >= o) incl += x;
        }
        __syncthreads();
        if (lane == 31) run->w[warp] = incl;
        __syncthreads();
        long long before = 0;
        total = 0;
        for (int w = 0; w < NT / 32; w++) {
            if (w == warp) before = total;
            total += run->w[w];
        }
        return before + incl - mine;
    };
    long long mine = 0, total, round;
    for (int s = tid; s < a.slots; s += NT) mine += pt_units<NB>(a, s, tpb);
    const long long at = scan(mine, total);
    per = max((total * a.K + gridDim.x - 1) / gridDim.x, (long long)PT_LEAST);
    const long long from = blockIdx.x * per;
    left = max(0ll, min(per, total * a.K - from));
    auto found = [&](int s, long long before, long long units) {
        if (units > 0 && before * a.K <= from && from < (before + units) * a.K) {
            run->slot = s;
            run->off = from - before * a.K;
        }
    };
    if (a.slots <= NT) {
        found(tid, at, mine);
    } else if (left > 0) {  // the same for all threads
        long long before = 0;
        for (int s0 = 0; s0 < a.slots; s0 += NT) {
            const long long u = s0 + tid < a.slots ? pt_units<NB>(a, s0 + tid, tpb) : 0;
            const long long x = scan(u, round);
            found(s0 + tid, before + x, u);
            before += round;
        }
    }
}

// T: __half, __nv_bfloat16, or float for pairs.
template <typename T, int HD>
__global__ void __launch_bounds__(PtShape<HD, sizeof(T) == 4>::THREADS, 1)
    k_prompt_tc(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PromptArgs a,
                int tpb, int items) {
    constexpr bool PAIR = sizeof(T) == 4, BF = std::is_same<T, __nv_bfloat16>::value;
    typedef PtShape<HD, PAIR> Z;
    constexpr int NB = Z::NB, SB = Z::SB, HALVES = Z::HALVES, COLS = Z::COLS, STAGE = Z::STAGE;
    constexpr int STAGES = Z::STAGES, TCOLS = Z::TCOLS, WARPS = Z::WARPS;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t* s_q = sm;  // [NB][HD / 64][128][128]
    uint8_t* ring = sm + NB * Z::QBLOCK;
    PtBars<NB>* bars = (PtBars<NB>*)(ring + STAGES * STAGE);
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
            mbar_init(&bars->item_empty[s], 3 + WARPS);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&bars->q_full[b], 1);
            mbar_init(&bars->q_empty[b], 1);
            mbar_init(&bars->s_full[b], 1);
            mbar_init(&bars->p_half[b], 8);
            mbar_init(&bars->p_full[b], 8);
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
    long long per = 0, left = 0;
    if (a.cut) pt_run<NB, Z::THREADS>(a, tpb, &bars->run, per, left);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem = bars->tmem;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return pt_wait(bar, parity, &bars->failed, a.status);
    };
    auto all = [&](uint64_t* bar, uint32_t parity) {  // the same answer for the warp
        return __all_sync(FULL, wait(bar, parity)) != 0;
    };
    // the item that every role works on, in the same order, held until `done`; null: no more
    int n_item = 0;
    auto next = [&]() -> const PtItem<NB>* {
        const int s = n_item % PT_RING;
        if (!all(&bars->item_full[s], n_item / PT_RING)) return nullptr;
        return bars->item[s].more ? &bars->item[s] : nullptr;
    };
    auto done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->item_empty[n_item % PT_RING]);
        n_item++;
    };
    constexpr TtTile tile = {1024, PT_KEYS * 128};
    TtPlace at = {0, 0};
    const int halves = PAIR ? 2 : HALVES == 1 || a.D <= 128 ? 1 : HALVES;
    // columns of 64 dims that half h of a row has
    auto cols_of = [&](int h) { return PAIR ? (a.D + 63) / 64 : min(COLS, (a.D - h * 128 + 63) / 64); };

    if (warp >= WARPS) {
    if (warp == WARPS) {  // ---- copies
        int q_count[2] = {0, 0};
        int filled = 0, asks = 0;  // stages filled so far, V tiles to be looked over
        bool ok = true;
        if (tt_elect()) {
            tma_prefetch_desc(&map_q);
            tma_prefetch_desc(&map_k);
            tma_prefetch_desc(&map_v);
        }
        __syncwarp();
        int head = 0, key0 = 0;
        auto load = [&](const CUtensorMap* map, int i) {  // keys of tile i
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                if (h >= halves) continue;
                const int s = at.stage;
                if (filled >= STAGES) ok = ok && all(&bars->empty[s], at.phase ^ 1);
                if (ok && tt_elect()) {
                    const int cols = cols_of(h);
                    mbar_expect_tx(&bars->full[s], cols * PT_KEYS * 128);
                    for (int c = 0; c < cols; c++)
                        tt_copy_q(ring + s * STAGE + c * PT_KEYS * 128, map, h * Z::WIDTH + c * 64,
                                  head, key0 + i * PT_KEYS, &bars->full[s]);
                }
                __syncwarp();
                filled += ok;
                if (ok) at.next(STAGES);
            }
        };
        while (const PtItem<NB>* x = ok ? next() : nullptr) {
            const PtTiles<NB> t = x->t;
            head = x->head;
            key0 = x->it.key0;
            const int row0 = x->it.row0;
            done();
            if (t.lo >= t.hi) continue;
            load(&map_k, t.lo);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (t.b[b].lo >= t.b[b].hi) continue;
                if (q_count[b] > 0) ok = ok && all(&bars->q_empty[b], q_count[b] - 1);
                if (ok && tt_elect()) {
                    int cols = 0;
                    for (int h = 0; h < halves; h++) cols += cols_of(h);
                    mbar_expect_tx(&bars->q_full[b], cols * tpb * a.G * 128);
                    for (int h = 0; h < halves; h++)
                        for (int c = 0; c < cols_of(h); c++)
                            tt_copy_q(s_q + b * Z::QBLOCK + (h * COLS + c) * Z::QCOL, &map_q,
                                      h * Z::WIDTH + c * 64, head * a.G, row0 + b * tpb,
                                      &bars->q_full[b]);
                }
                __syncwarp();
                q_count[b] += ok;
            }
            for (int i = t.lo; i < t.hi && ok; i++) {
                if (NB == 1 && i + 1 < t.hi) load(&map_k, i + 1);
                load(&map_v, i);
                if (!PAIR && t.look(i)) {
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
    } else if (warp == WARPS + 1) {  // ---- products: one elected lane
        constexpr uint32_t id_s = tt_idesc<BF>(PT_KEYS, false, false);
        const uint64_t q0 = umma_desc_sw128(smem_addr(s_q)), kv0 = tt_desc(smem_addr(ring), tile);
        const int steps = (a.D + 15) / 16;
        const uint32_t id_o[2] = {tt_idesc<BF>(min(128, (a.D + 15) & ~15), false, true),
                                  tt_idesc<BF>(max(16, (a.D - 128 + 15) & ~15), false, true)};
        if (tt_elect()) {
        int n[2] = {0, 0}, q_count[2] = {0, 0};  // tiles and items of each row block
        bool ok = true;
        while (ok) {
            const int slot = n_item % PT_RING;
            if (!wait(&bars->item_full[slot], n_item / PT_RING)) break;
            if (!bars->item[slot].more) break;
            const PtTiles<NB> t = bars->item[slot].t;
            mbar_arrive(&bars->item_empty[slot]);
            n_item++;
            // S = Q K^T of row block b, tile i, whose K is at place k
            auto scores = [&](int b, int i, const TtPlace& k) {
                const int m = n[b] + i - t.b[b].lo, sb = NB == 2 ? b : m & 1;
                if (i == t.b[b].lo) ok = ok && wait(&bars->q_full[b], q_count[b]++);
                const uint32_t d = tmem + b * TCOLS + (NB == 2 ? 0 : sb * PT_KEYS);
                TtPlace x = k;
                // half h of q's columns times the stage at place x
                auto product = [&](int h, const TtPlace& x, uint32_t more, bool low) {
                    const uint64_t dk = kv0 + ((x.stage * STAGE) >> 4);
                    const uint64_t dq = q0 + ((b * Z::QBLOCK + h * COLS * Z::QCOL) >> 4);
#pragma unroll
                    for (int s = 0; s < COLS * 4; s++)
                        if ((PAIR ? 0 : h * 8) + s < steps) {
                            const uint64_t sq = dq + (((s >> 2) * Z::QCOL + (s & 3) * 32) >> 4);
                            const uint64_t sk = dk + (((s >> 2) * tile.col + (s & 3) * 32) >> 4);
                            if (PAIR && low && s == 0) pt_mma_ss_low(d, sq, sk, id_s);
                            else umma_f16(d, sq, sk, id_s, s > 0 ? 1u : more);
                        }
                };
#pragma unroll
                for (int h = 0; h < HALVES; h++) {
                    if (h >= halves) continue;
                    ok = ok && wait(&bars->full[x.stage], x.phase);
                    tc_fence_after();
                    // pairs: low parts of q times the high ones of k, high ones of q times the
                    // low ones of k, both 2^PT_LOW too large, and the high ones of both last,
                    // since a sum is cut at each step by what it has grown to
                    if (ok) product(PAIR ? 1 - h : h, x, h > 0, false);
                    x.next(STAGES);
                }
                if (PAIR && ok) product(0, k, 1, true);
                if (!ok) return;
                tc_commit(&bars->s_full[sb]);
                if (i + 1 == t.b[b].hi) tc_commit(&bars->q_empty[b]);
            };
            // O += P V of row block b, tile i, whose V is at place v
            auto values = [&](int b, int i, const TtPlace& v) {
                const int m = n[b] + i - t.b[b].lo, sb = NB == 2 ? b : m & 1;
                TtPlace x = v;
                for (int h = 0; h < halves; h++, x.next(STAGES))
                    ok = ok && wait(&bars->full[x.stage], x.phase);
                const uint32_t p = tmem + b * TCOLS + (NB == 2 ? 0 : sb * PT_KEYS);
                const uint32_t o = tmem + b * TCOLS + SB * PT_KEYS + (PAIR ? (m & 1) * HD : 0);
                const uint32_t before = !PAIR && i > t.b[b].lo;  // (pairs: a tile's sums alone)
                bool skip = false;
#pragma unroll
                for (int part = 0; part < 2; part++) {
                    ok = ok && wait(part ? &bars->p_full[sb] : &bars->p_half[sb], NB == 2 ? m : m >> 1);
                    tc_fence_after();
                    if (!PAIR && part == 0 && t.b[b].mixed(i)) skip = *(volatile uint32_t*)&bars->skip[sb];
                    if (!ok || skip) continue;
                    x = v;
#pragma unroll
                    for (int h = 0; h < HALVES; h++) {
                        if (h >= halves) continue;
                        const uint64_t dv = kv0 + ((x.stage * STAGE) >> 4);
#pragma unroll
                        for (int y = 0; y < 4; y++) {  // 32 keys of each half of the tile
                            const int s = (y >> 1) * 4 + (1 - part) * 2 + (y & 1);
                            const uint64_t ds = dv + ((s * 2 * tile.group) >> 4);
                            // pairs: low weights times high values, high weights times low ones
                            pt_mma_ts(PAIR ? o : o + h * 128,
                                      p + (s >> 2) * (PT_KEYS / 2) + (s & 3) * 8 +
                                          (PAIR && h == 0 ? 32 : 0),
                                      ds, id_o[PAIR ? 0 : h],
                                      part + y + (PAIR ? h : 0) > 0 ? 1u : before);
                        }
                        x.next(STAGES);
                    }
                    if (PAIR && part) {  // high times high last, as for the scores
                        const uint64_t dv = kv0 + ((v.stage * STAGE) >> 4);
                        pt_mma_ts_low(o, p, dv, id_o[0]);
#pragma unroll
                        for (int s = 1; s < PT_KEYS / 16; s++)
                            pt_mma_ts(o, p + (s >> 2) * (PT_KEYS / 2) + (s & 3) * 8,
                                      dv + ((s * 2 * tile.group) >> 4), id_o[0], 1);
                    }
                }
                if (ok) tc_commit(&bars->pv[PAIR ? m & 1 : b]);
            };
            auto release = [&](TtPlace& x) {  // a K or V tile, by the products issued so far
                for (int h = 0; h < halves; h++, x.next(STAGES))
                    if (ok) tc_commit(&bars->empty[x.stage]);
            };
            if (t.lo < t.hi) {
#pragma unroll
                for (int b = 0; b < NB; b++)
                    if (t.b[b].in(t.lo)) scores(b, t.lo, at);
                release(at);
            }
#pragma unroll 1
            for (int i = t.lo; i < t.hi && ok; i++) {
                const bool more = i + 1 < t.hi;
                if (NB == 1) {
                    if (more) {
                        scores(0, i + 1, at);
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
                        if (more && t.b[b].in(i + 1)) scores(b, i + 1, k);
                    }
                    if (more) release(at);
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b++) n[b] += t.b[b].hi - t.b[b].lo;
        }
        // every product issued has ended before the block frees its TMEM
        tc_commit(&bars->done);
        (void)mbar_wait(&bars->done, 0, TT_WAIT_NS);
        }
        __syncwarp();
    } else if (warp == WARPS + 2) {  // ---- which item comes next
        if (blockIdx.x == 0) prompt_check(a, lane, 32);
        int count = 0;
        auto give = [&](const PtItem<NB>& x) {
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
        bool ok = true;
        PtItem<NB> p;
        p.more = 1;
        p.slot = 0;
        // the item's head, and whether there is work for it here
        auto ready = [&](int head) {
            p.head = head;
            if (!PAIR) return true;
            const uint32_t* m = a.amax + ((size_t)p.it.req * a.K + head) * PR_MAGS;
            p.k_back = exp2f((float)-pr_shift(m[PR_K]));
            p.v_back = exp2f((float)-pr_shift(m[PR_V]));
            return !pr_odd(a, p.it.req, head);
        };
        if (!a.cut) {  // whole items, long ones first; every second round of the CTAs goes back
            p.whole = 1;
            for (int round = 0; ok && round * (int)gridDim.x < items; round++) {
                const int c = round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
                const int x = round * gridDim.x + c;
                if (x >= items) continue;
                p.it = prompt_item(a, a.slots - 1 - x / a.K);
                if (p.it.rows <= 0 || !ready(x % a.K)) continue;
                p.t.set(a, p.it, tpb);
                ok = give(p);
            }
        } else {
            PromptPiece cut = {};
            int slot = left > 0 ? bars->run.slot : a.slots, u = 0, head = 0, pos = 0;
            long long at = blockIdx.x * per;  // unit of the item's tile `pos`
            auto open = [&]() {               // the next slot with rows, from `slot`
                for (; slot < a.slots; slot++) {
                    p.it = prompt_item(a, slot);
                    if (p.it.rows > 0) break;
                }
                if (slot >= a.slots) return;
                p.t.set(a, p.it, tpb);
                u = p.t.hi - p.t.lo + PT_PAD;
            };
            open();
            if (left > 0 && u > 0) {
                head = (int)(bars->run.off / u);
                pos = (int)(bars->run.off - (long long)head * u);
            }
            while (ok && left > 0 && slot < a.slots) {
                const int tiles = u - PT_PAD;
                const bool cuts = tiles >= PT_CUT;
                const int n = cuts ? (int)min((long long)(tiles - pos), left) : tiles;
                // (an item that is not cut is its first unit's CTA's)
                if (ready(head) && (cuts ? n > 0 : pos == 0)) {
                    PtItem<NB> x = p;
                    x.whole = n == tiles;
                    x.slot = at == blockIdx.x * per ? 0 : 1;
                    if (!x.whole) {
                        x.t.clip(p.t.lo + pos, p.t.lo + pos + n);
                        if (pos == 0)
                            cut = {p.it.row0, p.it.rows, head,
                                   (int)((at + tiles - 1) / per - blockIdx.x) + 1, x.slot};
                    }
                    ok = give(x);
                }
                at += u - pos;
                left -= u - pos;
                pos = 0;
                if (++head == a.K) {
                    head = 0;
                    slot++;
                    open();
                }
            }
            if (lane == 0) a.pieces[blockIdx.x] = cut;
        }
        PtItem<NB> end = {};
        if (ok) give(end);
    } else {  // ---- values that are not finite, in mixed tiles
        int looks = 0;
        uint32_t used = 0;  // stages before this item
        bool ok = true;
        while (const PtItem<NB>* item = ok ? next() : nullptr) {
            const PtTiles<NB> t = item->t;
            done();
            // (pairs are finite: what was not is zero)
            const int last = PAIR ? t.lo : t.hi;
            for (int i = t.lo; i < last && ok; i++) {
                if (i == t.all0 && i < t.all1) i = t.all1;
                if (i >= t.hi) break;
                uint32_t bits = 0;
                constexpr uint32_t e = BF ? 0x7f807f80u : 0x7c007c00u;
                constexpr uint32_t one = BF ? 0x00800080u : 0x04000400u;
                TtPlace x = pt_place<STAGES>(used + t.before(i) * halves);
                // asked for once the stage's copy before is over: its phase cannot be taken
                // for the one before, and the stage is held until P is there
                ok = all(&bars->ask[looks % PT_LOOKS], looks / PT_LOOKS);
                for (int h = 0; h < halves && ok; h++, x.next(STAGES)) {
                    ok = all(&bars->full[x.stage], x.phase);
                    const uint8_t* v = ring + x.stage * STAGE;
                    const int n = cols_of(h) * PT_KEYS * 128;
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
            used += 2 * (t.hi - t.lo) * halves;
        }
    }
    } else {  // ---- softmax: two threads to a row, half of a tile's keys each
        const int b = warp >> 3, half = warp >> 2 & 1, m = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + b * TCOLS + ((uint32_t)(warp & 3) << 21);
        const uint32_t t_o = lanes + SB * PT_KEYS;
        const float log2e = 1.44269504088896341f;
        // the reference lies LIFT below the largest score that it was taken from, which may
        // grow by GROWN before the sums are rescaled: weights stay below 2^15.  Of pairs the
        // heaviest is 2^13 at least, so that the others lose at most 2^-49 of it
        constexpr float LIFT = PAIR ? 13.f : TT_LIFT<BF>, GROWN = PAIR ? 2.f : 8.f;
        const bool cap = a.softcap > 0.f;
        const float c0 = cap ? log2e : a.scale * log2e;
        const float y0 = cap ? 2.f * log2e * a.scale / a.softcap : 0.f;
        const int tok = b * tpb + m / a.G;  // of the item
        const bool mine = m < tpb * a.G;
        // a wait that gives up sets `failed`: later ones return at once, and the next item
        // is the last
        auto pass = [&](uint64_t* bar, uint32_t parity) {
            (void)wait(bar, parity);
            __syncwarp();
            tc_fence_after();
        };
        // the row's two warps meet
        auto meet = [&]() {
            asm volatile("bar.sync %0, 64;" ::"r"(1 + b * 4 + (warp & 3)) : "memory");
        };
        int n = 0, looks = 0;
        uint32_t used = 0;  // stages before this item
        while (true) {
            // both of the row's warps or neither: after a wait that gave up one may be without
            const PtItem<NB>* x = next();
            uint32_t both;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                "bar.red.and.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                : "=r"(both)
                : "r"((uint32_t)(x != nullptr)), "r"(1 + b * 4 + (warp & 3))
                : "memory");
            if (!both) break;
            const PtBlock blk = x->t.b[b];
            const bool row = mine && tok < x->it.rows;
            const bool work = __any_sync(FULL, row);  // the same for the row's two warps
            // the row sees keys [low, lim]
            auto lim = [&]() { return row ? min(x->it.past + tok, x->it.keys - 1) : -1; };
            auto low = [&]() { return a.window > 0 ? max(0, x->it.past + tok - a.window + 1) : 0; };
            float back = 1.f;  // pairs: what the row's scores were divided by
            if (PAIR && row)
                back = x->k_back * a.q_back[(long long)(x->it.row0 + tok) * a.H + x->head * a.G +
                                            m - m / a.G * a.G];
            // (not 0, however small q and k: scores of -inf stay -inf)
            const float c2 = PAIR && !cap ? fmaxf(c0 * back, 0x1p-126f) : c0;
            // running maximum of the scores, the weights' reference (in powers of two),
            // and the sum of this thread's weights
            float top = -INFINITY, ref = -INFINITY, sum = 0.f;
            // pairs: half of the row's sums.  The tensor cores cut their f32 sums, which over
            // many tiles shows (4096 keys: 7e-6), so each tile's are added here
            [[maybe_unused]] float acc[PAIR ? HD / 2 : 1], late = 1.f;  // late: for the tile not added yet
            [[maybe_unused]] auto add = [&](int tile_n) {
                pass(&bars->pv[tile_n & 1], tile_n >> 1);
#pragma unroll
                for (int c = 0; c < HD / 2; c += 16) {
                    uint32_t o[16];
                    tt_load<16>(t_o + (tile_n & 1) * HD + half * (HD / 2) + c, o);
#pragma unroll
                    for (int j = 0; j < 16; j++) acc[c + j] = fmaf(__uint_as_float(o[j]), late, acc[c + j]);
                }
                late = 1.f;
            };
            if constexpr (PAIR) {
#pragma unroll
                for (int c = 0; c < HD / 2; c++) acc[c] = 0.f;
            }
#pragma unroll 1
            for (int i = blk.lo; i < blk.hi; i++, n++) {
                const int sb = NB == 2 ? b : n & 1, kt = i * PT_KEYS;
                const bool mixed = blk.mixed(i);
                const uint32_t t_s = lanes + (NB == 2 ? 0 : sb * PT_KEYS);
                float s[32], from = 0.f;  // scores of 32 keys
                const uint32_t t_h = t_s + half * (PT_KEYS / 2);
                pass(&bars->s_full[sb], NB == 2 ? n : n >> 1);
                if (work) {
                    // rare work on the scores in place, by calls: the code of every tile is
                    // then fetched without jumps over it (16384 bf16 tokens: 2.04 ms with it
                    // in line, 1.88 without it)
                    if (cap && PAIR) pt_cap_f32(t_h, a.softcap, back * a.scale / a.softcap);
                    else if (cap) pt_cap(t_h, a.softcap, y0);
                    if (mixed) pt_hide(t_h, low() - kt - half * 64, lim() - kt - half * 64);
                    float t0 = top, t1 = top, t2 = top, t3 = top;
                    auto largest = [&]() {
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            t0 = pt_max3(t0, s[j], s[j + 1]);
                            t1 = pt_max3(t1, s[j + 2], s[j + 3]);
                            t2 = pt_max3(t2, s[j + 4], s[j + 5]);
                            t3 = pt_max3(t3, s[j + 6], s[j + 7]);
                        }
                    };
                    tt_load<32>(t_h, (uint32_t*)s);
                    largest();
                    tt_load<32>(t_h + 32, (uint32_t*)s);
                    largest();
                    top = pt_max3(pt_max3(t0, t1, t2), t3, t3);
                    // a buffer of its own for each row block, or for each of two tiles
                    // running: it is written again when the other thread has read it
                    float(*at)[128] = bars->meet[sb];
                    at[half][m] = top;
                    tc_fence_before();
                    meet();
                    tc_fence_after();
                    top = pt_max3(top, at[half ^ 1][m], top);
                    const float want = top == -INFINITY ? -INFINITY : top * c2 - LIFT;
                    if (i == blk.lo) {
                        ref = want;
                    } else if (__any_sync(FULL, row && !(want - ref <= GROWN) && want != -INFINITY)) {
                        const float fix = ref == -INFINITY ? 0.f : tt_exp2(ref - want);
                        // O holds the tiles so far (two row blocks: since the scores came)
                        if (NB == 1 && !PAIR) pass(&bars->pv[b], n - 1);
                        sum *= fix;
                        ref = want;
                        if constexpr (PAIR) {
                            late = fix;
#pragma unroll
                            for (int c = 0; c < HD / 2; c++) acc[c] *= fix;
                        }
#pragma unroll 1
                        for (int c = PAIR ? a.D : half * 16; c < a.D; c += 32) {
                            uint32_t o[16];
                            tt_load<16>(t_o + c, o);
#pragma unroll
                            for (int j = 0; j < 16; j++)
                                o[j] = __float_as_uint(__uint_as_float(o[j]) * fix);
                            tt_st<16>(t_o + c, o);
                        }
                    }
                    // a reference that is not finite makes every weight NaN
                    from = ref == -INFINITY ? 0.f : ref + (ref - ref);
                }
                float l[4] = {};
                auto weights = [&](int c) {  // of keys c .. c + 31 of the half, over its scores
                    uint32_t p[16], low[16];
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float y0 = tt_exp2(fmaf(s[j], c2, -from));
                        const float y1 = tt_exp2(fmaf(s[j + 1], c2, -from));
                        l[j & 3] += y0;
                        l[j & 3 | 1] += y1;
                        p[j >> 1] = pt_pack<BF>(y0, y1);
                        if constexpr (PAIR) {
                            const float2 h = __half22float2(*(const __half2*)&p[j >> 1]);
                            constexpr float up = 1 << PT_LOW;
                            low[j >> 1] = pt_pack<BF>((y0 - h.x) * up, (y1 - h.y) * up);
                        }
                    }
                    // the second 32 keys come first, whose weights may go over the first ones'
                    // scores when those have been read again (kept, 96 registers a thread
                    // were not enough)
                    if (c > 0) tt_load<32>(t_h, (uint32_t*)s);
                    tt_st<16>(t_h + c / 2, p);
                    if constexpr (PAIR) tt_st<16>(t_h + 32 + c / 2, low);
                    tt_wait_st();
                };
                if (work) weights(32);
                bool odd = false;
                if (mixed && !PAIR) {
                    const int y = looks + x->t.looks(i);
                    pass(&bars->look[y % PT_LOOKS], y / PT_LOOKS);
                    odd = *(volatile uint32_t*)&bars->odd[y % PT_LOOKS];
                    if ((warp & 7) == 0 && lane == 0) bars->skip[sb] = odd;
                }
                // the product starts when half of the weights are there
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->p_half[sb]);
                if (work) {
                    weights(0);
                    sum += (l[0] + l[1]) + (l[2] + l[3]);
                }
                if (!PAIR && odd) {
                    const uint8_t* vt[2];
                    TtPlace at = pt_place<STAGES>(used + x->t.before(i) * halves);
                    for (int h = 0; h < halves; h++, at.next(STAGES)) {
                        pass(&bars->full[at.stage], at.phase);
                        vt[h] = ring + at.stage * STAGE;
                    }
                    if (i > blk.lo) pass(&bars->pv[b], n - 1);
                    tc_fence_before();
                    meet();  // the weights of both halves are there
                    tc_fence_after();
                    if (work)
                        pt_careful<BF>(t_s, t_o, vt, a.D, half, low() - kt, lim() - kt,
                                       i == blk.lo);
                }
                // with two buffers of scores the product before may still run: the item's end
                // waits for this tile's by parity, which must not take the phase before for it
                if (NB == 1 && !PAIR && i > blk.lo && i + 1 == blk.hi) pass(&bars->pv[b], n - 1);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->p_full[sb]);
                if constexpr (PAIR)
                    if (work && i > blk.lo) add(n - 1);
            }
            looks += x->t.looks(x->t.hi);
            used += 2 * (x->t.hi - x->t.lo) * halves;
            // ---- the item's end
            const bool none = blk.lo >= blk.hi;
            if (!none) {
                if constexpr (PAIR) add(n - 1);
                else pass(&bars->pv[b], n - 1);
                if (work) {
                    float(*at)[128] = bars->meet[NB == 2 ? b : 0];
                    at[half][m] = sum;
                    meet();
                    sum += at[half ^ 1][m];
                    meet();  // read before the next item's first tile
                }
            }
            const int row0 = x->it.row0, head = x->head;
            const bool whole = x->whole;
            const size_t piece = ((size_t)blockIdx.x * 2 + x->slot) * (NB * 128) + b * 128 + m;
            const float v_back = PAIR ? x->v_back : 1.f;
            done();
            if (!work) continue;
            const int g = m - m / a.G * a.G;  // query head of the kv head
            if (!whole) {  // the partial state
                if (half == 0) a.ml[piece] = make_float2(ref, none ? -1.f : sum);
                if (none) continue;
                float* to = a.part + piece * a.dp;
                if constexpr (PAIR) {
#pragma unroll
                    for (int c = 0; c < HD / 2; c += 8) {
                        const int d = half * (HD / 2) + c;
#pragma unroll
                        for (int j = 0; j < 8; j++) acc[c + j] *= v_back;
                        if (d < a.dp) pt_store32(to + d, (const uint32_t*)acc + c);
                    }
                } else {
#pragma unroll 1
                    for (int c = half * 16; c < a.D; c += 32) {
                        uint32_t o[16];
                        __syncwarp();
                        tt_load<16>(t_o + c, o);
                        pt_store32(to + c, o);
                        if (c + 8 < a.D) pt_store32(to + c + 8, o + 8);
                    }
                }
                __syncwarp();
                tc_fence_before();
                continue;
            }
            const float inv = (sum > 0.f || sum != sum ? 1.f / sum : 0.f) * v_back;
            T* out = (T*)a.out + ((long long)(row0 + tok) * a.H + head * a.G + g) * a.D;
            const bool wide = ((uintptr_t)out & 31) == 0 && (a.D & 15) == 0;
            if constexpr (PAIR) {
                if (row) {
#pragma unroll
                    for (int c = 0; c < HD / 2; c += 8) {
                        const int d = half * (HD / 2) + c;
#pragma unroll
                        for (int j = 0; j < 8; j++) acc[c + j] = inv == 0.f ? 0.f : acc[c + j] * inv;
                        if (wide && d < a.D) pt_store32(out + d, (const uint32_t*)acc + c);
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (!wide && d + j < a.D) out[d + j] = acc[c + j];
                    }
                }
            } else {
#pragma unroll 1
                for (int c = half * 16; c < a.D; c += 32) {
                    uint32_t o[16], w[8];
                    __syncwarp();
                    if (!none) tt_load<16>(t_o + c, o);
                    if (!row) continue;
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        w[j] = none || inv == 0.f
                                   ? 0u
                                   : pt_pack<BF>(__uint_as_float(o[2 * j]) * inv,
                                                 __uint_as_float(o[2 * j + 1]) * inv);
                    if (wide) {
                        pt_store32(out + c, w);
                    } else {
                        *(uint4*)(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                        if (c + 8 < a.D) *(uint4*)(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
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

// Joins the pieces of the items that a run's end cut, a warp per row.
constexpr int PJ_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(PJ_WARPS * 32)
    k_prompt_join(const __grid_constant__ PromptArgs a, int tpb, int rows) {
    pdl_trigger();
    pdl_wait();
    const PromptPiece p = a.pieces[blockIdx.x];
    const int m = blockIdx.y * PJ_WARPS + (threadIdx.x >> 5);
    const int r = m & 127, tok = (m >> 7) * tpb + r / a.G;
    if (p.count <= 1 || r >= tpb * a.G || tok >= p.rows) return;
    T* out = (T*)a.out + ((long long)(p.row0 + tok) * a.H + p.head * a.G + r - r / a.G * a.G) * a.D;
    prompt_join_row(a, p.count, out, [&](int i) {
        return ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? p.slot : 0)) * rows + m;
    });
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

// Rows of `heads` heads as [rows][heads][dims], boxes of 64 dims (zeros past the last) by
// `box_heads` heads by `box_rows` rows.
static int pt_map(CUtensorMap* map, const void* base, bool bf, int dims_, int heads, int rows,
                  long long stride, int box_heads, int box_rows) {
    auto enc = pt_encode_fn();
    CW_CHECK(enc, CW_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    if (rows == 1) stride = (long long)heads * dims_;  // not used, and may be anything
    cuuint64_t dims[3] = {(cuuint64_t)dims_, (cuuint64_t)heads, (cuuint64_t)rows};
    cuuint64_t strides[2] = {(cuuint64_t)dims_ * 2, (cuuint64_t)stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                     const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CW_CHECK(r == CUDA_SUCCESS, CW_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return CW_OK;
}

// ---- f32 operands as pairs ---------------------------------------------------------
// x 2^s = h + l to 22 bits, h and l 2^PT_LOW f16, s by request and kv head (k, v) or by row and
// head (q).  With the largest in [2^14, 2^15), what is dropped is at most 2^-50 of the largest,
// or 2^-22 of the value itself (what that asks of the values: PR_APART).  A warp takes a head
// row, or for the magnitudes 32 of them.  4096 tokens of 16/8 heads of 128: 28 us for the
// magnitudes and 36 for the pairs of 252 (cold launches; 171 are the attention's, 6.5 the f32
// kernel's look at what is left to it); both wait for their reads.
constexpr int PS_WARPS = 8;
constexpr int PS_ROWS = 8;  // rows of a warp in flight

// The request whose rows [starts[r], starts[r + 1]) hold row t, or -1.
__device__ __forceinline__ int ps_req(const int* starts, int n_req, int t) {
    int lo = 0, hi = n_req;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return starts[lo] <= t && t < starts[lo + 1] ? lo : -1;
}
__global__ void __launch_bounds__(PS_WARPS * 32) k_prompt_amax(const __grid_constant__ PromptArgs a) {
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * PS_WARPS + (threadIdx.x >> 5);
    const int heads = 2 * a.K, head = (int)(w % heads), t0 = (int)(w / heads) * 32;
    pdl_wait();
    pdl_trigger();
    if (t0 >= a.n_keys) return;
    const bool is_v = head >= a.K;
    const int h = is_v ? head - a.K : head;
    const float* x = (const float*)(is_v ? a.v : a.k) + (long long)h * a.D;
    const long long stride = is_v ? a.v_stride : a.k_stride;
    const int* ks = a.key_starts ? a.key_starts : a.starts;
    uint32_t most = 0, least = ~0u;
    int mine = -1;
    auto flush = [&]() {
        if (lane == 0 && mine >= 0 && most) {
            uint32_t* m = a.amax + ((size_t)mine * a.K + h) * PR_MAGS;
            atomicMax(&m[is_v ? PR_V : PR_K], most);
            atomicMax(&m[is_v ? PR_V_LEAST : PR_K_LEAST], ~least);
        }
        most = 0;
        least = ~0u;
    };
    // several rows at a time: their reads are in flight together
    for (int t = t0; t < min(t0 + 32, a.n_keys); t += PS_ROWS) {
        uint32_t row[PS_ROWS] = {};
#pragma unroll
        for (int u = 0; u < PS_ROWS; u++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (t + u < a.n_keys && e * 32 + lane < a.D)
                    row[u] = max(row[u], __float_as_uint(fabsf(x[(t + u) * stride + e * 32 + lane])));
#pragma unroll
        for (int u = 0; u < PS_ROWS; u++) {
            if (t + u >= a.n_keys) break;
            const uint32_t r = __reduce_max_sync(FULL, row[u]);
            if (mine < 0 || t + u >= ks[mine + 1]) {
                flush();
                mine = ps_req(ks, a.n_req, t + u);
            }
            if (mine < 0 || r == 0) continue;
            most = max(most, r);
            least = min(least, r);
        }
    }
    flush();
}
// out: q, then k, then v, as [rows][heads][h: W, l: W] f16, zeros past D.
template <int W>
__global__ void __launch_bounds__(PS_WARPS * 32)
    k_prompt_pairs(const __grid_constant__ PromptArgs a, __half* out) {
    constexpr int N = W / 32;
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * PS_WARPS + (threadIdx.x >> 5);
    const long long nq = (long long)a.n_rows * a.H, nk = (long long)a.n_keys * a.K;
    if (w >= nq + 2 * nk) return;
    pdl_wait();
    pdl_trigger();
    const int kind = w < nq ? 0 : w < nq + nk ? 1 : 2;
    const long long i = kind == 0 ? w : kind == 1 ? w - nq : w - nq - nk;
    const int heads = kind == 0 ? a.H : a.K, t = (int)(i / heads), h = (int)(i - (long long)t * heads);
    const float* src = (const float*)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                       t * (kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride) +
                       (long long)h * a.D;
    const int req = ps_req(kind == 0 || !a.key_starts ? a.starts : a.key_starts, a.n_req, t);
    float x[N];
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < N; e++) {
        x[e] = lane * N + e < a.D && req >= 0 ? src[lane * N + e] : 0.f;
        most = max(most, __float_as_uint(fabsf(x[e])));
    }
    uint32_t* m = req >= 0 ? a.amax + ((size_t)req * a.K + (kind == 0 ? h / a.G : h)) * PR_MAGS : nullptr;
    if (kind == 0) {
        most = __reduce_max_sync(FULL, most);
        if (lane == 0) {
            if (pr_misfit(most) && m) atomicMax(&m[PR_Q], PR_ODD);
            a.q_back[i] = exp2f((float)-pr_shift(most));
        }
    } else {
        most = m ? m[kind == 1 ? PR_K : PR_V] : 0;
    }
    const float by = exp2f((float)pr_shift(most));
    __half hi[N], lo[N];
#pragma unroll
    for (int e = 0; e < N; e++) {
        float y = x[e] * by;
        if (!(fabsf(y) < 65504.f)) y = 0.f;  // not used: the f32 kernel's
        hi[e] = __float2half_rn(y);
        lo[e] = __float2half_rn((y - __half2float(hi[e])) * (1 << PT_LOW));
    }
    __half* to = out + w * 2 * W + lane * N;
    if constexpr (N == 4) {
        *(uint2*)to = *(const uint2*)hi;
        *(uint2*)(to + W) = *(const uint2*)lo;
    } else {
        *(uint32_t*)to = *(const uint32_t*)hi;
        *(uint32_t*)(to + W) = *(const uint32_t*)lo;
    }
}

bool prompt_tc_takes(const PromptArgs& a, uint32_t type) {
    if (a.G > 128 || !(a.scale > 0.f)) return false;
    if (type == CW_GGUF_F32)
        // Any place and stride; the pairs are laid out anew.  Short requests are faster on the
        // f32 kernel, and so are few rows over many keys, whose pairs are formed for little (us
        // there and here, heads of 128: with 16/8 heads a prompt of 128 tokens 28 and 33, of 192
        // 39 and 35, 32 of 64 47 and 79, 32 of 128 125 and 129; eight rows after 500 keys each 27
        // and 62, 32 after 300 53 and 119, 128 times four after 1000 650 and 1130, a row after
        // 1000 57 and 46, after 4000 54 and 64, 16 after 4000 62 and 65; with 32/8 heads 32 prompts
        // of 128 219 and 191, with 4/2 heads 42 and 54; 128 rows after 1000 645 and 1110 with
        // either 16/8 or 32/8 heads, 167 and 312 with 4/2).  The lengths are means, all that the
        // host knows: 4096 tokens beside 30 requests of one token take 2090 there and 300
        // here.  (Requests told apart on the device ended that, but the launches that then found
        // nothing made even batches slower: 32 prompts of 64 47 and 68, 128 of 16 48 and 70.)
        return a.D <= 128 && (long long)a.n_keys >= 160ll * a.n_req &&
               (a.n_rows >= 8ll * a.n_req || (a.n_req == 1 && a.n_keys < 2000));
    const long long strides = (a.n_rows > 1 ? a.q_stride : 0) |
                              (a.n_keys > 1 ? a.k_stride | a.v_stride : 0);
    return a.D % 8 == 0 && strides % 8 == 0 &&
           (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0;
}

template <typename T, int HD> static int pt_go(cw_ctx* ctx, PromptArgs& a) {
    constexpr bool PAIR = sizeof(T) == 4, BF = std::is_same<T, __nv_bfloat16>::value;
    typedef PtShape<HD, PAIR> Z;
    auto kern = k_prompt_tc<T, HD>;
    const int tpb = 128 / a.G;  // tokens of a row block
    a.bt = Z::NB * tpb;
    a.slots = a.n_rows / a.bt + a.n_req;
    const long long items = (long long)a.slots * a.K;
    CW_CHECK(items < (1ll << 30), CW_ERR_UNSUPPORTED, "cw_prompt_attention: too many rows");
    // Whole items or equal runs, from what the host knows: the longest item, or rounds of the
    // mean one, against the tiles a CTA would have and 9 tiles' time for the second launch and
    // the partial states (us, whole and cut: one prompt of 1024 rows 27 and 37, 2048 rows 49
    // and 70; four pieces of 270 rows after 6000 209 and 158, a row after 16000 209 and 31).
    const double rows = (double)a.n_rows / a.n_req, keys = (double)a.n_keys / a.n_req;
    const double work = a.K * (double)a.n_req * std::ceil(rows / a.bt), sms = ctx->sm_count;
    const double longest = keys / PT_KEYS, mean = std::max(keys - rows / 2, 1.0) / PT_KEYS;
    a.cut = std::max(longest, std::ceil(work / sms) * mean) > work * (mean + PT_PAD) / sms + 9.0;
    const int grid = a.cut ? ctx->sm_count : (int)std::min<long long>(items, ctx->sm_count);
    a.dp = (a.D + 7) / 8 * 8;
    constexpr int ROWS = Z::NB * 128;
    size_t need = 0;
    auto take = [&](size_t n) {  // a part of the scratch, at a multiple of 256
        const size_t at = need;
        need += (n + 255) / 256 * 256;
        return at;
    };
    const size_t pieces = a.cut ? (size_t)grid * 2 * ROWS : 0;
    const size_t at_part = take(pieces * a.dp * 4), at_ml = take(pieces * 8),
                 at_pieces = take(a.cut ? grid * sizeof(PromptPiece) : 0);
    char* base = nullptr;
    auto scratch = [&]() -> int {
        if (!need) return CW_OK;
        CW_TRY(stream_scratch(ctx, &ctx->prompt_scratch, &ctx->prompt_scratch_bytes, need,
                              "cw_prompt_attention"));
        base = (char*)ctx->prompt_scratch;
        a.part = (float*)(base + at_part);
        a.ml = (float2*)(base + at_ml);
        a.pieces = (PromptPiece*)(base + at_pieces);
        return CW_OK;
    };
    CUtensorMap mq, mk, mv;
    if constexpr (PAIR) {
        const size_t nq = (size_t)a.n_rows * a.H, nk = (size_t)a.n_keys * a.K;
        const size_t most = (size_t)a.n_req * a.K * PR_MAGS * 4;
        const size_t at_pairs = take((nq + 2 * nk) * 2 * HD * 2), at_back = take(nq * 4),
                     at_most = take(most);
        CW_TRY(scratch());
        __half* out = (__half*)(base + at_pairs);
        a.q_back = (float*)(base + at_back);
        a.amax = (uint32_t*)(base + at_most);
        CW_CUDA(cudaMemsetAsync(a.amax, 0, most, ctx->stream));
        const size_t b0 = ((size_t)(a.n_keys + 31) / 32 * 2 * a.K + PS_WARPS - 1) / PS_WARPS;
        const size_t b1 = (nq + 2 * nk + PS_WARPS - 1) / PS_WARPS;
        CW_CHECK(b1 < (1ull << 31), CW_ERR_UNSUPPORTED, "cw_prompt_attention: too many rows");
        CW_TRY(launch_pdl(ctx, false, k_prompt_amax, dim3((unsigned)b0), dim3(PS_WARPS * 32), 0, a));
        CW_TRY(launch_pdl(ctx, true, k_prompt_pairs<HD>, dim3((unsigned)b1), dim3(PS_WARPS * 32), 0,
                          a, out));
        CW_TRY(pt_map(&mq, out, false, 2 * HD, a.H, a.n_rows, 2ll * HD * a.H, a.G, tpb));
        CW_TRY(pt_map(&mk, out + nq * 2 * HD, false, 2 * HD, a.K, a.n_keys, 2ll * HD * a.K, 1, PT_KEYS));
        CW_TRY(pt_map(&mv, out + (nq + nk) * 2 * HD, false, 2 * HD, a.K, a.n_keys, 2ll * HD * a.K, 1,
                      PT_KEYS));
    } else {
        CW_TRY(scratch());
        CW_TRY(pt_map(&mq, a.q, BF, a.D, a.H, a.n_rows, a.q_stride, a.G, tpb));
        CW_TRY(pt_map(&mk, a.k, BF, a.D, a.K, a.n_keys, a.k_stride, 1, PT_KEYS));
        CW_TRY(pt_map(&mv, a.v, BF, a.D, a.K, a.n_keys, a.v_stride, 1, PT_KEYS));
    }
    static bool set[64] = {};
    if (!set[ctx->device & 63]) {
        CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)Z::SMEM));
        set[ctx->device & 63] = true;
    }
    CW_TRY(launch_pdl(ctx, true, kern, dim3(grid), dim3(Z::THREADS), Z::SMEM, mq, mk, mv, a, tpb,
                      (int)items));
    if (a.cut)
        CW_TRY(launch_pdl(ctx, true, k_prompt_join<T>, dim3(grid, ROWS / PJ_WARPS), dim3(PJ_WARPS * 32), 0,
                          a, tpb, ROWS));
    return check_launch("prompt_attention");
}
template <typename T> static int pt_dims(cw_ctx* ctx, PromptArgs& a) {
    if (a.D <= 64) return pt_go<T, 64>(ctx, a);
    if constexpr (sizeof(T) == 2)
        if (a.D > 128) return pt_go<T, 256>(ctx, a);
    return pt_go<T, 128>(ctx, a);
}
int prompt_tc_launch(cw_ctx* ctx, PromptArgs& a, uint32_t type) {
    if (type == CW_GGUF_F32) return pt_dims<float>(ctx, a);
    return type == CW_GGUF_BF16 ? pt_dims<__nv_bfloat16>(ctx, a) : pt_dims<__half>(ctx, a);
}

}  // namespace cw
