// cw_tree_tc.cuh -- what the tcgen05 kernels of cw_tree_attention share: TMEM loads
// and stores, the layout of a K or V tile in shared memory, the ring of tiles and the
// warp that fills it.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "cw_gemm.cuh"
#include "cw_tree.cuh"

namespace cw {

constexpr int TT_STAGES = 16;  // most stages of the ring (one K or V tile each)
constexpr uint64_t TT_WAIT_NS = 2000000000ull;
// Weights are powers of two over a reference, rounded to the cache's type.  In f16 the
// reference is 2^7 below the scores it was taken from: the largest weight is then 2^7 to
// 2^15 and those down to 2^-31 of it are kept (2^-24 before; 30000 keys e^-17.5 of one
// other lost their joint share, 7.5e-4 of the result).
template <bool BF> constexpr float TT_LIFT = BF ? 0.f : 7.f;

__device__ __forceinline__ void tt_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tt_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
template <int N> __device__ __forceinline__ void tt_st(uint32_t addr, const uint32_t* r) {
    if constexpr (N == 32) {
        tt_st32(addr, r);
    } else if constexpr (N == 16) {
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
            "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
            "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
            "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
            "r"(r[15])
            : "memory");
    } else {
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr),
            "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
            : "memory");
    }
}
// Waits for this thread's TMEM loads; the values pass through, so no use of them can
// be moved before it.
__device__ __forceinline__ void tt_wait_ld32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                   "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tt_wait_ld16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tt_ld8(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7])::"memory");
}
// N columns, waited for.
template <int N> __device__ __forceinline__ void tt_load(uint32_t addr, uint32_t* r) {
    if constexpr (N == 64) {
        tt_ld32(addr, r);
        tt_ld32(addr + 32, r + 32);
        tt_wait_ld32(r);
        tt_wait_ld32(r + 32);
    } else if constexpr (N == 32) {
        tt_ld32(addr, r);
        tt_wait_ld32(r);
    } else if constexpr (N == 8) {
        tt_ld8(addr, r);
    } else {
        tmem_ld16(addr, *(uint32_t(*)[16])r);
        tt_wait_ld16(r);
    }
}
__device__ __forceinline__ uint32_t tt_ld1(uint32_t addr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void tt_st1(uint32_t addr, uint32_t r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(addr), "r"(r)
                 : "memory");
}
__device__ __forceinline__ void tt_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tt_fence_async() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// D[tmem] += A[tmem] B[shared], in the TMEM lanes whose bits in off0 (lanes 0-31) ..
// off3 (lanes 96-127) are 0.
__device__ __forceinline__ void tt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                          uint32_t off0, uint32_t off1, uint32_t off2,
                                          uint32_t off3) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 1, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%4, %5, %6, %7}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(off0), "r"(off1), "r"(off2), "r"(off3)
        : "memory");
}
// How a K or V tile lies in shared memory: 1024-byte atoms of 8 keys x 64 dims
// (128-byte swizzled), `group` bytes from 8 keys to the next and `col` bytes from 64
// dims to the next.  Where D fills the instance's columns (tt_wide) one copy brings all
// of a page's rows and dims, atoms of 8 keys side by side; else a copy per 64 dims, and
// those past D read zeros.
__host__ __device__ constexpr bool tt_wide(int D) { return D == 64 || D == 128 || D == 256; }
struct TtTile {
    uint32_t group, col;
    __device__ __forceinline__ uint32_t at(int key, int chunk) const {  // 16-byte chunk
        return (key >> 3) * group + (chunk >> 3) * col + (key & 7) * 128 +
               (((chunk ^ key) & 7) << 4);
    }
};
// Matrix descriptors of such a tile: contraction over dims (K), where the column
// step is not used, and over keys (V).
__device__ __forceinline__ uint64_t tt_desc(uint32_t saddr, const TtTile& t) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(t.col >> 4) << 16) |
           ((uint64_t)(t.group >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tt_copy(void* dst, const CUtensorMap* map, int x, int group,
                                        uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %3, %4}], [%5];" ::"r"(smem_addr(dst)),
        "l"((uint64_t)map), "r"(x), "r"(0), "r"(group), "r"(smem_addr(bar))
        : "memory");
}
// 64 dims from x of a box of query rows: heads from `head`, tokens from `row`.
__device__ __forceinline__ void tt_copy_q(void* dst, const CUtensorMap* map, int x, int head,
                                          int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_addr(dst)),
        "l"((uint64_t)map), "r"(x), "r"(head), "r"(row), "r"(smem_addr(bar))
        : "memory");
}
// Instruction descriptor: 128 x n, f32 sums; a_rows, b_rows: the operand's contraction
// index is the row in memory.
template <bool BF>
__host__ __device__ constexpr uint32_t tt_idesc(int n, bool a_rows, bool b_rows) {
    return (1u << 4) | (BF ? (1u << 7) | (1u << 10) : 0u) | (a_rows ? 1u << 15 : 0u) |
           (b_rows ? 1u << 16 : 0u) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ float tt_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Two weights rounded and packed (first in the low half), their rounded values added.
template <bool BF> __device__ __forceinline__ uint32_t tt_pack(float x, float y, float& sum) {
    uint32_t r;
    if (BF) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
        sum += __uint_as_float(r << 16) + __uint_as_float(r & 0xffff0000u);
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
        const float2 f = __half22float2(*(const __half2*)&r);
        sum += f.x + f.y;
    }
    return r;
}
template <bool BF> __device__ __forceinline__ float tt_value(uint32_t bits16) {
    if (BF) return __uint_as_float(bits16 << 16);
    return __half2float(__ushort_as_half((unsigned short)bits16));
}
template <bool BF> __device__ __forceinline__ bool tt_odd(uint32_t bits16) {
    const uint32_t e = BF ? 0x7f80u : 0x7c00u;
    return (bits16 & e) == e;
}
template <bool BF> __device__ __forceinline__ bool tt_odd8(const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; i++) odd |= tt_odd<BF>(w[i] & 0xffffu) | tt_odd<BF>(w[i] >> 16);
    return odd;
}
// A place in the ring.  An item's tiles pass through it as K0, V0, K1, V1, .. or, with
// two buffers of scores, as K0, then K(i+1), V(i) in turn.
struct TtPlace {
    int stage;
    uint32_t phase;
    __device__ __forceinline__ void next(int stages) {
        if (++stage == stages) {
            stage = 0;
            phase ^= 1;
        }
    }
    __device__ __forceinline__ void skip(int n, int stages) {
        stage += n;
        while (stage >= stages) {
            stage -= stages;
            phase ^= 1;
        }
    }
};
__device__ __forceinline__ bool tt_elect() {  // one lane of a converged warp
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r != 0;
}

// Fills the ring from the pages of an item: one warp, all lanes, a copy each.  A stage
// holds SK keys of K or of V.
template <int COLS, int SK> struct TtFeed {
    static constexpr int STAGE = COLS * SK * 128;
    const TreeArgs& a;
    uint8_t* ring;
    uint64_t *full, *empty;
    uint32_t* lost;
    const int stages, lane;
    TtPlace at = {0, 0};
    bool filled = false;  // every stage has been filled once
    // the lane's copy of a stage: `box` keys (a page, or 64 of a larger one) from key
    // pi * box, dims from 64 * col
    int box, boxes, pi, col, shift;
    uint32_t box_bytes, dst;
    // the item: its pages from page0's first key on, 32 ids to a read and a read ahead
    const int* ids;
    int in0, last, pages, head, have, now_ids, next_ids;
    int first;            // key of the item, counted like `last`, that rows may see first

    __device__ TtFeed(const TreeArgs& a_, uint8_t* ring_, uint64_t* full_, uint64_t* empty_,
                      uint32_t* lost_, int stages_, const TtTile& t)
        : a(a_), ring(ring_), full(full_), empty(empty_), lost(lost_), stages(stages_),
          lane(threadIdx.x & 31) {
        const bool wide = tt_wide(a.D);
        box = min(a.page, 64);
        const int per = SK / box;
        boxes = wide ? per : per * COLS;
        pi = lane % per;
        col = lane / per;
        box_bytes = box * 128 * (wide ? COLS : 1);
        dst = pi * (box >> 3) * t.group + col * t.col;
        shift = (a.page & (a.page - 1)) == 0 ? __ffs(a.page) - 1 : -1;
    }
    __device__ int read(int j) const { return j + lane < pages ? ids[j + lane] : -1; }
    __device__ void begin(const TreeItem& it) {
        const int key0 = (it.q.tile0 + it.tile) * TR_TILE, page0 = key0 / a.page;
        in0 = key0 - page0 * a.page;
        last = min(it.q.keys - key0, it.tiles * TR_TILE);  // keys of this piece
        first = tree_first(a, it.q) - key0;
        pages = (in0 + last + a.page - 1) / a.page;
        ids = a.table + (size_t)it.r * a.max_pages + page0;
        head = it.head;
        have = 0;
        now_ids = read(0);
        next_ids = read(32);
    }
    // The lane's copy of the item's keys [j * SK, ..+SK) as the cache's 8-row group; -1:
    // none, -2: keys without a page, -3: and a row may see some of them.
    __device__ int place(int j) {
        const int off = in0 + j * SK + pi * box;
        const int p = shift >= 0 ? off >> shift : off / a.page;
        if (__shfl_sync(FULL, p, 0) - have >= 32) {
            have += 32;
            now_ids = next_ids;
            next_ids = read(have + 32);
        }
        const int x = __shfl_sync(FULL, now_ids, p & 31);
        const int y = __shfl_sync(FULL, next_ids, p & 31);
        if (lane >= boxes || j * SK + pi * box >= last) return -1;
        const int id = p - have < 32 ? x : y;
        if (id < 0 || id >= a.n_pages) return j * SK + (pi + 1) * box > first ? -3 : -2;
        return ((id * a.K + head) * a.page + (off - p * a.page)) >> 3;
    }
    // Keys without a page: zeros in place of an old tile.
    static __device__ __noinline__ void lack(uint8_t* to, uint32_t bytes, uint32_t* lost,
                                             int* status) {
        for (uint32_t i = 0; i < bytes; i += 16) *(uint4*)(to + i) = make_uint4(0, 0, 0, 0);
        tt_fence_async();
        if (!lost) return;
        *(volatile uint32_t*)lost = 1;  // the weight warps look at ids from here on
        atomicCAS(status, DEV_OK, DEV_BAD_INPUT);
    }
    // Into the next stage once it is free; all(bar, parity) waits, the warp together.
    template <typename All> __device__ bool load(const CUtensorMap* map, int group, All all) {
        const int s = at.stage;
        if (filled && !all(&empty[s], at.phase ^ 1)) return false;
        const uint32_t live = __popc(__ballot_sync(FULL, group >= 0));
        if (group < -1)  // rare, and a call (256 x 1 at 3001: 206 us, 217 with its code here)
            lack(ring + s * STAGE + dst, box_bytes, group == -3 ? lost : nullptr, a.status);
        __syncwarp();
        // copies may count before these bytes are announced: the phase lacks lane 0's arrival
        if (lane == 0) mbar_expect_tx(&full[s], live * box_bytes);
        if (group >= 0) tt_copy(ring + s * STAGE + dst, map, col * 64, group, &full[s]);
        at.next(stages);
        filled |= at.stage == 0;
        return true;
    }
    // After a wait that gave up: copies in flight land before the block may end.
    __device__ void drain() const {
        for (int s = 0; s < stages; s++)
            if (filled || s < at.stage)  // the last filling of stage s
                (void)mbar_wait(&full[s], s < at.stage ? at.phase : at.phase ^ 1, TT_WAIT_NS);
    }
};

// A wait that gives up sets `failed`, and later waits return at once: the TMA and MMA
// loops end, the softmax warps (which meet at barriers) run through their items
// without waiting.
__device__ __forceinline__ bool tt_wait(uint64_t* bar, uint32_t parity, uint32_t* failed,
                                        int* status) {
    if (mbar_try_wait(bar, parity & 1)) return true;
    if (*(volatile uint32_t*)failed) return false;
    const uint64_t from = global_ns();
    do {
        for (int i = 0; i < 256; i++)  // reading the clock would delay the wake-up
            if (mbar_try_wait(bar, parity & 1)) return true;
    } while (global_ns() - from < TT_WAIT_NS);
    gm_fail(status);
    *(volatile uint32_t*)failed = 1;
    return false;
}

// cw_tree_tc.cu: the cache's tensor map.  cw_tree_few.cu: the kernel of short row blocks.
int tt_map(CUtensorMap* map, const void* base, const TreeArgs& a, bool bf);
int tt_map_q(CUtensorMap* map, const TreeArgs& a, bool bf);
bool tt_few_takes(const TreeArgs& a);
int tt_few_launch(cw_ctx* ctx, const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv,
                  bool bf, int grid);

}  // namespace cw
