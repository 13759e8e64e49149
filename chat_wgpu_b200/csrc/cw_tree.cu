// cw_tree.cu -- cw_tree_attention: the kernel for f32 caches and for shapes that
// the tcgen05 kernels (cw_tree_few.cu, cw_tree_tc.cu) do not take, and the launch that
// joins the pieces of cut items.
//
//   s = scale * q . k,  s' = softcap tanh(s / softcap),  o = sum p v / sum p,
//   p = exp(s' - running maximum) over the keys the row sees.
//
// f32 accuracy on the warp-level tensor cores: every f32 operand x is the sum of
// two TF32 values, x = h + l to within 2^-21 |x|, and a product is h h' + h l' + l h'
// with f32 sums (the dropped l l' is below 2^-21 of the product).
// 16-bit operands are exact in one TF32 value, so their l terms are left out.
//
// Block: 8 warps, WM groups of 16 rows by WK = 8 / WM groups of 64 / WK keys; each
// warp keeps its rows' maximum, sum and weighted values over its own keys, joined
// through shared memory at the item's end.  K and V tiles go through a ring of
// cp.async buffers, 16-byte chunks exclusive-ored with the row so that the
// fragment loads below are free of bank conflicts.  The contraction order is free,
// so thread (g, t) of a warp takes the head dims 8t..8t+7 of each 32 (two 16-byte
// loads per row) and key pair 2t, 2t+1 of each 8: the accumulator layout of the
// scores is then the operand layout of the weights, with no exchange.
//
// Bound by the products and the splits: 8 requests x 24 nodes (64-row blocks) at 4500
// take 7.3 us a 64-key tile, 3.4 us of it the TF32 rate of mma.sync; the bytes alone
// would take 1.5 us.  One token at 1037 takes 15 us, the latency of its dependent reads
// (lengths, page ids, one tile) and of the joining launch.
#include <math.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "cw_tree.cuh"

namespace cw {

constexpr int TR_THREADS = 256;
constexpr int TR_ROWS = 2;  // tiles whose row offsets are kept
constexpr int TR_HAVE = 8;  // tiles whose sets of keys with a page are kept (the ring's 4 and more)
constexpr size_t TR_SMEM_CAP = 226 * 1024 + 384;  // dynamic; the kernel also has static

__device__ __forceinline__ void tr_cp16(void* dst, const void* src, bool live) {
    const int n = live ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(dst)),
                 "l"(src), "r"(n)
                 : "memory");
}
__device__ __forceinline__ void tr_cp4(void* dst, const void* src, bool live) {
    const int n = live ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(dst)),
                 "l"(src), "r"(n)
                 : "memory");
}
__device__ __forceinline__ void tr_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void tr_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// x = h + l: h cut to TF32's 10 bits, l = x - h (exact) rounded to them, so h + l is
// within 2^-21 of x.  Whole-number operations: the conversion instruction runs at a
// fraction of their rate (8 x 24 f32 nodes at 4500: 232 us with it throughout, 205
// without).  Infinities keep l = 0, NaN keeps h.
__device__ __forceinline__ uint32_t tr_low(float x, uint32_t h) {
    return (__float_as_uint(x - __uint_as_float(h)) + 0x1000u) & 0xffffe000u;
}
__device__ __forceinline__ void tr_split(float x, uint32_t& h, uint32_t& l) {
    h = __float_as_uint(x) & 0xffffe000u;
    l = tr_low(x, h);
}
// The same with h rounded, so that l is as often below zero as above.  One operand of a
// product is split this way: cut on both sides, the dropped l l' would all have the
// product's sign and scale the scores by about 1 - 2^-22.
__device__ __forceinline__ void tr_split_even(float x, uint32_t& h, uint32_t& l) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(h) : "f"(x));
    l = tr_low(x, h);
}
__device__ __forceinline__ void tr_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16-byte chunk c of row j in a swizzled tile of DP floats a row.
template <int DP> __device__ __forceinline__ int tr_at(int j, int c) {
    return j * DP + ((c & ~7) | ((c ^ j) & 7)) * 4;
}

// Ring buffers (one K or V tile each) that fit beside the queries.
template <int DP, int BM> constexpr int tr_ring() {
    const size_t left = TR_SMEM_CAP - (size_t)BM * DP * 4 - BM * 8 - TR_ROWS * TR_TILE * 8 - 1024;
    const size_t n = left / ((size_t)TR_TILE * DP * 4);
    return n > 8 ? 8 : (int)n;
}
template <int DP, int BM> constexpr size_t tr_smem() {
    return ((size_t)tr_ring<DP, BM>() * TR_TILE + BM) * DP * 4 + (size_t)BM * 8  // sees
           + TR_ROWS * TR_TILE * 8                                              // row offsets
           + 128 * 8;                                                           // warp max, sum
}

// An item once more, from f32 products: what the pairs cannot say.  A part of a pair times
// an infinity can be NaN where the whole product is not (0 or the other sign in its low
// part), so an item whose sums are NaN ends here, whichever way they came about.  Leaves
// the weighted values in key group 0 of `so` (zeros in the others) and each row's
// reference and sum in s_sees.  All threads; out of line, its registers are its own.
template <typename T, int DP, int BM>
__device__ __noinline__ void tr_careful(const TreeArgs& a, TreeItem it, float* so, const float* sq,
                                        uint64_t* s_sees) {
    float* sx = so + 128 * DP;  // [BM][64] scores, then weights
    float* s_fix = sx + BM * TR_TILE;
    const int tid = threadIdx.x;
    const float c2 = a.softcap > 0.f ? 1.44269504088896341f : a.scale * 1.44269504088896341f;
    float top = -INFINITY, rf = -INFINITY, sum = 0.f;  // thread m: of row m, as in k_tree
    for (int i = tid; i < 128 * DP; i += TR_THREADS) so[i] = 0.f;
#pragma unroll 1
    for (int t = 0; t < it.tiles; t++) {
        const int kt = (it.q.tile0 + it.tile + t) * TR_TILE;
        auto at = [&](int j) {  // a seen key's row in the cache
            const int pi = (kt + j) / a.page;
            return (((long long)a.table[(size_t)it.r * a.max_pages + pi] * a.K + it.head) * a.page +
                    (kt + j - pi * a.page)) * a.D;
        };
        if (tid < it.rows) {
            uint64_t see = tree_sees(a, it.q, it.block * BM + tid, kt);
            for (uint64_t left = see; left; left &= left - 1) {
                const int j = __ffsll((long long)left) - 1;
                if (!tree_has(a, it.r, kt + j)) see &= ~(1ull << j);
            }
            s_sees[tid] = see;
        }
        __syncthreads();
        for (int i = tid; i < it.rows * TR_TILE; i += TR_THREADS) {
            const int m = i / TR_TILE, j = i % TR_TILE;
            float x = -INFINITY;
            if (s_sees[m] >> j & 1) {
                const T* k = (const T*)a.k + at(j);
                x = 0.f;
                for (int d = 0; d < a.D; d++)
                    x = fmaf(sq[tr_at<DP>(m, d >> 2) + (d & 3)], tree_f32<T>(k[d]), x);
                if (a.softcap > 0.f) x = a.softcap * tanhf(x * a.scale / a.softcap);
            }
            sx[i] = x;
        }
        __syncthreads();
        if (tid < it.rows) {
            float* x = sx + tid * TR_TILE;
            for (int j = 0; j < TR_TILE; j++) top = fmaxf(top, x[j]);
            const float ref = top == -INFINITY ? 0.f : __fmul_rn(top, c2);
            const float fix = rf == -INFINITY ? 0.f : exp2f(rf - ref);
            sum *= fix;
            for (int j = 0; j < TR_TILE; j++) {
                x[j] = exp2f(fmaf(x[j], c2, -ref));
                sum += x[j];
            }
            rf = top == -INFINITY ? -INFINITY : ref;
            s_fix[tid] = fix;
        }
        __syncthreads();
        for (int i = tid; i < it.rows * a.D; i += TR_THREADS) {
            const int m = i / a.D, d = i - m * a.D;
            float* o = so + tr_at<DP>(m, d >> 2) + (d & 3);
            float x = *o * s_fix[m];
            for (uint64_t left = s_sees[m]; left; left &= left - 1) {
                const int j = __ffsll((long long)left) - 1;
                x = fmaf(sx[m * TR_TILE + j], tree_f32<T>(((const T*)a.v)[at(j) + d]), x);
            }
            *o = x;
        }
        __syncthreads();
    }
    if (tid < BM) ((float2*)s_sees)[tid] = make_float2(rf, sum);
    __syncthreads();
}

// VEC: rows and offsets allow 4-element vectors.
template <typename T, int DP, int WM, bool VEC>
__global__ void __launch_bounds__(TR_THREADS, 1) k_tree(const __grid_constant__ TreeArgs a) {
    constexpr int BM = 16 * WM, WK = 8 / WM, KW = TR_TILE / WK, NB = KW / 8, DB = DP / 32;
    constexpr int RING = tr_ring<DP, BM>();
    constexpr bool EXACT = sizeof(T) == 2;  // operands are TF32 values already
    static_assert(RING >= 3, "the ring holds a tile in use and two in flight");
    static_assert(RING * TR_TILE * DP >= 128 * DP + BM * TR_TILE + BM, "room for tr_careful");
    extern __shared__ __align__(16) float sm[];
    float* ring = sm;
    float* sq = ring + RING * TR_TILE * DP;
    uint64_t* s_sees = (uint64_t*)(sq + BM * DP);
    long long* s_row = (long long*)(s_sees + BM);  // [TR_ROWS][64] offset of a key row, or -1
    float2* s_ml = (float2*)(s_row + TR_ROWS * TR_TILE); // [WK][BM]
    __shared__ uint64_t s_have[TR_HAVE];  // [tile % TR_HAVE] keys whose page is in the cache
    __shared__ int s_edge;
    __shared__ TreeShared s_run;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int wm = warp % WM, wk = warp / WM, g = lane >> 2, t4 = lane & 3;
    pdl_wait();
    pdl_trigger();
    TreeRun run = tree_run<TR_THREADS>(a, &s_run);
    TreeItem it;
    bool any = false;
    while (run.left > 0) {
        it = tree_next(a, run);
        any = true;
        const T* kb = (const T*)a.k;
        const T* vb = (const T*)a.v;
        const int key0 = (it.q.tile0 + it.tile) * TR_TILE;
        const int m0 = it.block * BM;
        // ---- queries, and the window's edge
        if (tid == 0) s_edge = 0;
        __syncthreads();
        if (tid < BM && tid < it.rows) {
            const int e = tree_edge(a, it.q, m0 + tid);
            if (e > 0) atomicMax(&s_edge, e);
        }
        for (int i = tid; i < BM * (DP / 4); i += TR_THREADS) {
            const int m = i / (DP / 4), c = i % (DP / 4);
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            if (m < it.rows) {
                const int node = (m0 + m) / a.G, gi = (m0 + m) - node * a.G;
                const T* src = (const T*)a.q + (long long)(it.q.row0 + node) * a.q_stride +
                               (long long)(it.head * a.G + gi) * a.D + 4 * c;
                if (VEC && 4 * c < a.D) {
                    if constexpr (sizeof(T) == 4) {
                        const float4 f = *(const float4*)src;
                        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
                    } else {
                        const uint2 raw = *(const uint2*)src;
                        const T* e = (const T*)&raw;
                        for (int j = 0; j < 4; j++) x[j] = tree_f32<T>(e[j]);
                    }
                } else if (!VEC) {
                    for (int j = 0; j < 4; j++)
                        if (4 * c + j < a.D) x[j] = tree_f32<T>(src[j]);
                }
            }
            *(float4*)(sq + tr_at<DP>(m, c)) = make_float4(x[0], x[1], x[2], x[3]);
        }
        // ---- the ring: buffer s % RING holds K (s even) or V of tile s / 2
        const int steps = 2 * it.tiles;
        auto rows_of = [&](int tile) {  // threads 0..63: the tile's key rows in the cache
            if (tid >= TR_TILE) return;
            const int j = key0 + tile * TR_TILE + tid;
            long long at = -1;
            if (tile < it.tiles && j < it.q.keys) {
                const int pi = j / a.page;
                const int id = a.table[(size_t)it.r * a.max_pages + pi];
                if (id >= 0 && id < a.n_pages)
                    at = (((long long)id * a.K + it.head) * a.page + (j - pi * a.page)) * a.D;
                else if (j >= tree_first(a, it.q))
                    tree_bad(a);
            }
            s_row[(tile & 1) * TR_TILE + tid] = at;
            const uint32_t have = __ballot_sync(FULL, at >= 0);
            if (lane == 0) ((uint32_t*)&s_have[tile & (TR_HAVE - 1)])[warp] = have;
        };
        auto load = [&](int s) {
            if (s < steps) {
                const T* base = s & 1 ? vb : kb;
                float* dst = ring + (s % RING) * TR_TILE * DP;
                const long long* rows = s_row + ((s >> 1) & 1) * TR_TILE;
                for (int i = tid; i < TR_TILE * (DP / 4); i += TR_THREADS) {
                    const int j = i / (DP / 4), c = i % (DP / 4);
                    const long long at = rows[j];
                    float* d = dst + tr_at<DP>(j, c);
                    const T* src = base + (at < 0 ? 0 : at);
                    if constexpr (sizeof(T) == 4) {
                        if (VEC) {
                            const bool live = at >= 0 && 4 * c < a.D;
                            tr_cp16(d, live ? src + 4 * c : src, live);
                        } else {
                            for (int e = 0; e < 4; e++) {
                                const bool live = at >= 0 && 4 * c + e < a.D;
                                tr_cp4(d + e, live ? src + 4 * c + e : src, live);
                            }
                        }
                    } else {
                        float x[4] = {0.f, 0.f, 0.f, 0.f};
                        if (at >= 0 && VEC && 4 * c < a.D) {
                            const uint2 raw = *(const uint2*)(src + 4 * c);
                            const T* e = (const T*)&raw;
                            for (int k = 0; k < 4; k++) x[k] = tree_f32<T>(e[k]);
                        } else if (at >= 0 && !VEC) {
                            for (int k = 0; k < 4; k++)
                                if (4 * c + k < a.D) x[k] = tree_f32<T>(src[4 * c + k]);
                        }
                        *(float4*)d = make_float4(x[0], x[1], x[2], x[3]);
                    }
                }
            }
            tr_commit();
        };
        for (int s = 0; s < RING - 1; s++) {
            if (!(s & 1) && s < steps) {
                __syncthreads();
                rows_of(s >> 1);
                __syncthreads();
            }
            load(s);
        }
        if (!((RING - 1) & 1)) {  // step 0 loads the K tile of the next pair
            __syncthreads();
            rows_of((RING - 1) >> 1);
        }
        // mx: running maximum of the scores; rf: what the weights so far refer to, in powers
        // of two (-inf before any).  rf is kept, not formed again from mx: its rounding,
        // 2^-24 of some 20, has to be the same in the weights and in their rescale (8 x 24
        // nodes at 4500: error 4e-7 against 64 bits, 1.5e-6 with it formed again).
        float o[DB][4][4], mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
        float rf[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int b = 0; b < DB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[b][i][e] = 0.f;
        // this warp's keys of a tile's set, the first in bit 0
        auto own_bits = [&](const uint64_t* set) {
            return ((const uint32_t*)set)[wk * KW >> 5] >> (wk * KW & 31);
        };
        const float c2 = a.softcap > 0.f ? 1.44269504088896341f : a.scale * 1.44269504088896341f;
        float p[NB][4];
        for (int s = 0; s < steps; s++) {
            const int kt = key0 + (s >> 1) * TR_TILE;
            const bool part = tree_partial(it.q, s_edge, kt);
            if (!(s & 1) && part && tid < BM) s_sees[tid] = tree_sees(a, it.q, m0 + tid, kt);
            tr_wait<RING - 2>();
            __syncthreads();  // tile s is here, and everyone is done with tile s - 1
            const float* tile = ring + (s % RING) * TR_TILE * DP;
            if (!(s & 1)) {
                // ---- scores of this warp's 16 rows and KW keys
#pragma unroll
                for (int n = 0; n < NB; n++) p[n][0] = p[n][1] = p[n][2] = p[n][3] = 0.f;
#pragma unroll
                for (int b = 0; b < DB; b++) {
                    float qa[2][8];
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int i = 0; i < 2; i++)
                            *(float4*)&qa[h][4 * i] = *(const float4*)(
                                sq + tr_at<DP>(wm * 16 + g + 8 * h, b * 8 + t4 * 2 + i));
                    uint32_t ah[4][4], al[4][4];
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const float x = qa[h][2 * k + i];
                                if (EXACT) ah[k][h + 2 * i] = __float_as_uint(x);
                                else tr_split_even(x, ah[k][h + 2 * i], al[k][h + 2 * i]);
                            }
#pragma unroll
                    for (int n = 0; n < NB; n++) {
                        float kf[8];
                        const int j = wk * KW + n * 8 + g;
#pragma unroll
                        for (int i = 0; i < 2; i++)
                            *(float4*)&kf[4 * i] =
                                *(const float4*)(tile + tr_at<DP>(j, b * 8 + t4 * 2 + i));
                        // fresh sums for each 32 dims, joined by f32 additions: the
                        // tensor core's own running sum is cut, not rounded
                        float hh[4] = {}, hl[4] = {}, lh[4] = {};
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            if (EXACT) {
                                tr_mma(hh, ah[k], __float_as_uint(kf[2 * k]),
                                       __float_as_uint(kf[2 * k + 1]));
                            } else {
                                uint32_t h0, l0, h1, l1;
                                tr_split(kf[2 * k], h0, l0);
                                tr_split(kf[2 * k + 1], h1, l1);
                                tr_mma(hh, ah[k], h0, h1);
                                tr_mma(hl, ah[k], l0, l1);
                                tr_mma(lh, al[k], h0, h1);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            p[n][e] += EXACT ? hh[e] : hh[e] + (hl[e] + lh[e]);
                    }
                }
                // ---- weights; accumulator element e: row g + 8 (e / 2), key 2 t4 + e % 2
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t sees = own_bits(&s_have[(s >> 1) & (TR_HAVE - 1)]);
                    if (part) sees &= own_bits(&s_sees[wm * 16 + g + 8 * h]);
                    float top = mx[h];
#pragma unroll
                    for (int n = 0; n < NB; n++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            float x = p[n][2 * h + i];
                            if (a.softcap > 0.f) x = a.softcap * tanhf(x * a.scale / a.softcap);
                            if (!(sees >> (n * 8 + 2 * t4 + i) & 1)) x = -INFINITY;
                            p[n][2 * h + i] = x;
                            top = fmaxf(top, x);
                        }
                    top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
                    const float ref = top == -INFINITY ? 0.f : __fmul_rn(top, c2);
                    const float fix = rf[h] == -INFINITY ? 0.f : exp2f(rf[h] - ref);
                    float add = 0.f;
#pragma unroll
                    for (int n = 0; n < NB; n++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const float w = exp2f(fmaf(p[n][2 * h + i], c2, -ref));
                            p[n][2 * h + i] = w;
                            add += w;
                        }
                    sum[h] = sum[h] * fix + add;
                    mx[h] = top;
                    rf[h] = top == -INFINITY ? -INFINITY : ref;
                    if (fix != 1.f) {
#pragma unroll
                        for (int b = 0; b < DB; b++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                o[b][i][2 * h] *= fix;
                                o[b][i][2 * h + 1] *= fix;
                            }
                    }
                }
            } else {
                // ---- weighted values.  A weight of 0 times a value that is not finite
                // would reach rows that do not see the key, so a tile that rows see
                // differently is looked over first (keys past the end were zero-filled).
                bool odd = false;
                uint32_t see0 = 0, see1 = 0;
                if (part) {
                    // read before the vote: after it the next tile's sets may be written
                    see0 = own_bits(&s_sees[wm * 16 + g]);
                    see1 = own_bits(&s_sees[wm * 16 + g + 8]);
                    for (int i = tid; i < TR_TILE * DP; i += TR_THREADS)
                        odd |= !(fabsf(tile[i]) <= 3.402823466e38f);
                    odd = __syncthreads_or(odd);
                }
                if (!odd) {
                    uint32_t ph[NB][4], pl[NB][4];
#pragma unroll
                    for (int n = 0; n < NB; n++) {
                        // operand order: row g key 2t, row g+8 key 2t, then key 2t+1
                        tr_split_even(p[n][0], ph[n][0], pl[n][0]);
                        tr_split_even(p[n][2], ph[n][1], pl[n][1]);
                        tr_split_even(p[n][1], ph[n][2], pl[n][2]);
                        tr_split_even(p[n][3], ph[n][3], pl[n][3]);
                    }
#pragma unroll
                    for (int b = 0; b < DB; b++) {
                        float hh[4][4] = {}, lo[4][4] = {};  // fresh sums, as for the scores
#pragma unroll
                        for (int n = 0; n < NB; n++) {
                            const int j = wk * KW + n * 8 + 2 * t4;
                            float v0[4], v1[4];
                            *(float4*)v0 = *(const float4*)(tile + tr_at<DP>(j, b * 8 + g));
                            *(float4*)v1 = *(const float4*)(tile + tr_at<DP>(j + 1, b * 8 + g));
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                if (EXACT) {
                                    const uint32_t x = __float_as_uint(v0[i]),
                                                   y = __float_as_uint(v1[i]);
                                    tr_mma(hh[i], ph[n], x, y);
                                    tr_mma(lo[i], pl[n], x, y);
                                } else {
                                    uint32_t h0, l0, h1, l1;
                                    tr_split(v0[i], h0, l0);
                                    tr_split(v1[i], h1, l1);
                                    tr_mma(hh[i], ph[n], h0, h1);
                                    tr_mma(lo[i], ph[n], l0, l1);
                                    tr_mma(lo[i], pl[n], h0, h1);
                                }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[b][i][e] += hh[i][e] + lo[i][e];
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < NB; n++)
#pragma unroll
                        for (int kk = 0; kk < 8; kk++) {
                            const int from = (lane & ~3) | (kk >> 1);
                            const float w0 = __shfl_sync(FULL, p[n][kk & 1], from);
                            const float w1 = __shfl_sync(FULL, p[n][2 + (kk & 1)], from);
                            const int j = n * 8 + kk;
#pragma unroll
                            for (int b = 0; b < DB; b++)
#pragma unroll
                                for (int e = 0; e < 8; e++) {
                                    const float v = tile[tr_at<DP>(wk * KW + j,
                                                                   b * 8 + t4 * 2 + (e >> 2)) +
                                                         (e & 3)];
                                    float* d = &o[b][e & 3][e >> 2];
                                    if (see0 >> j & 1) d[0] = fmaf(w0, v, d[0]);
                                    if (see1 >> j & 1) d[2] = fmaf(w1, v, d[2]);
                                }
                        }
                }
            }
            // the buffer of tile s - 1 is free since this step's barrier
            load(s + RING - 1);
            if (!((s + RING) & 1)) rows_of((s + RING) >> 1);
        }
        tr_wait<0>();
        // sums of NaN: the item once more, but not for rows whose query holds a NaN
        uint32_t nan = 0;  // bit h: of row g + 8 h
#pragma unroll
        for (int h = 0; h < 2; h++) {
            bool odd = sum[h] != sum[h];
#pragma unroll
            for (int b = 0; b < DB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    odd |= o[b][i][2 * h] != o[b][i][2 * h] ||
                           o[b][i][2 * h + 1] != o[b][i][2 * h + 1];
            if (odd && wm * 16 + g + 8 * h < it.rows) nan |= 1u << h;
        }
        bool careful = __syncthreads_or(nan);
        if (careful) {
            for (int h = 0; h < 2; h++)
                for (int d = 0; d < DP && (nan >> h & 1); d++) {
                    const float x = sq[tr_at<DP>(wm * 16 + g + 8 * h, d >> 2) + (d & 3)];
                    if (x != x) nan &= ~(1u << h);
                }
            careful = __syncthreads_or(nan);
        }
        float* so = ring;  // [WK][BM][DP], the ring is idle
        float2* s_all = (float2*)s_sees;  // each row's maximum and sum
        if (careful) {
            tr_careful<T, DP, BM>(a, it, so, sq, s_sees);
        } else {
            // ---- join the WK key groups: weights from the maxima, then the sums in turn
#pragma unroll
            for (int h = 0; h < 2; h++) {
                sum[h] += __shfl_xor_sync(FULL, sum[h], 1);
                sum[h] += __shfl_xor_sync(FULL, sum[h], 2);
                if (t4 == 0) s_ml[wk * BM + wm * 16 + g + 8 * h] = make_float2(rf[h], sum[h]);
            }
            __syncthreads();
            float own[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int m = wm * 16 + g + 8 * h;
                float top = -INFINITY;
                for (int w = 0; w < WK; w++) top = fmaxf(top, s_ml[w * BM + m].x);
                const float x = s_ml[wk * BM + m].x;
                own[h] = x == -INFINITY ? 0.f : exp2f(x - top);
            }
#pragma unroll
            for (int b = 0; b < DB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {  // dims b * 32 + t4 * 8 + 4 i ..
                        const int m = wm * 16 + g + 8 * h;
                        *(float4*)(so + wk * BM * DP + tr_at<DP>(m, b * 8 + t4 * 2 + i)) =
                            make_float4(o[b][0][i + 2 * h] * own[h], o[b][1][i + 2 * h] * own[h],
                                        o[b][2][i + 2 * h] * own[h], o[b][3][i + 2 * h] * own[h]);
                    }
            if (tid < BM) {
                float top = -INFINITY, l = 0.f;
                for (int w = 0; w < WK; w++) top = fmaxf(top, s_ml[w * BM + tid].x);
                for (int w = 0; w < WK; w++) {
                    const float2 x = s_ml[w * BM + tid];
                    if (x.y != 0.f) l += x.y * exp2f(x.x - top);  // 0: saw nothing; NaN stays
                }
                s_all[tid] = make_float2(top, l);
            }
            __syncthreads();
        }
        const size_t piece = (size_t)blockIdx.x * 2 + tree_slot(run, it);
        for (int i = tid; i < it.rows * a.D; i += TR_THREADS) {
            const int m = i / a.D, d = i - m * a.D;
            const float l = s_all[m].y;
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < WK; w++) x += so[w * BM * DP + tr_at<DP>(m, d >> 2) + (d & 3)];
            if (it.whole) {
                const int node = (m0 + m) / a.G, gi = (m0 + m) - node * a.G;
                ((T*)a.out)[((long long)(it.q.row0 + node) * a.H + it.head * a.G + gi) * a.D + d] =
                    tree_to<T>(l > 0.f || l != l ? x / l : 0.f);
            } else {
                a.part[(piece * BM + m) * a.dp + d] = x;
                if (d == 0) a.ml[piece * BM + m] = s_all[m];
            }
        }
        __syncthreads();
    }
    if (tid == 0) tree_record(a, run, it, any);
}

// Joins the pieces of the items that a run's end cut: out = sum_i w_i o_i / sum_i w_i
// l_i, w_i = 2^(m_i - max m), in key order.  A warp per row and 128 dims, 8 warps a
// block; bound by the latency of three dependent reads, so a lane has the four dims of
// eight pieces in flight.
constexpr int TJ_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(TJ_WARPS * 32) k_tree_join(const __grid_constant__ TreeArgs a) {
    pdl_trigger();  // the next call may set itself up; it waits for this one before it reads
    pdl_wait();
    const TreePiece p = a.pieces[blockIdx.x];
    const int lane = threadIdx.x & 31, m = blockIdx.y * TJ_WARPS + (threadIdx.x >> 5);
    const int d = blockIdx.z * 128 + 4 * lane;
    if (p.count <= 1 || m >= p.rows) return;
    auto piece = [&](int i) {
        return ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? p.slot : 0)) * a.bm + m;
    };
    float top = -INFINITY;
    for (int i = lane; i < p.count; i += 32) top = fmaxf(top, __ldcg(&a.ml[piece(i)]).x);
    top = warp_max(top);
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < p.count; i0 += 32) {
        float w = 0.f;
        if (i0 + lane < p.count) {
            const float2 x = __ldcg(&a.ml[piece(i0 + lane)]);
            if (x.y != 0.f) {  // 0: the row saw nothing there; NaN stays
                w = exp2f(x.x - top);
                l += w * x.y;
            }
        }
        const int n = min(32, p.count - i0);
        for (int j0 = 0; j0 < n; j0 += 8) {
            float4 x[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = j0 + j < n && d < a.D
                           ? __ldcg((const float4*)(a.part + piece(i0 + j0 + j) * a.dp + d))
                           : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float wj = __shfl_sync(FULL, w, (j0 + j) & 31);
                if (j0 + j >= n) continue;  // 0 times a NaN stays: keys of no weight, not finite
                acc.x = fmaf(wj, x[j].x, acc.x);
                acc.y = fmaf(wj, x[j].y, acc.y);
                acc.z = fmaf(wj, x[j].z, acc.z);
                acc.w = fmaf(wj, x[j].w, acc.w);
            }
        }
    }
    l = warp_sum(l);
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const int r = p.block * a.bm + m, node = r / a.G, gi = r - node * a.G;
    T* out = (T*)a.out + ((long long)(p.row0 + node) * a.H + p.head * a.G + gi) * a.D + d;
    const float y[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (d + e < a.D) out[e] = tree_to<T>(inv == 0.f ? 0.f : y[e] * inv);
}

// The context's scratch of at least `need` bytes, in stream order (no wait).  It comes
// from a pool of the process, which keeps what a context gives back: the partial states
// of a grid are up to 39 MB, and a plain allocation of that takes longer than the call.
// An outgrown block stays until the context goes, since a graph captured before may still
// write there; a new block is twice the old one at least, so they add up to less than it.
static int tree_scratch(cw_ctx* ctx, size_t need) {
    if (need <= ctx->tree_scratch_bytes) return CW_OK;
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    CW_CUDA(cudaStreamIsCapturing(ctx->stream, &cs));
    CW_CHECK(cs == cudaStreamCaptureStatusNone, CW_ERR_UNSUPPORTED,
             "cw_tree_attention: call once with these sizes before a stream capture");
    static std::mutex lock;
    static cudaMemPool_t pools[64] = {};
    CW_CHECK(ctx->device < 64, CW_ERR_UNSUPPORTED, "cw_tree_attention: device %d", ctx->device);
    cudaMemPool_t pool;
    {
        std::lock_guard<std::mutex> hold(lock);
        if (!pools[ctx->device]) {
            cudaMemPoolProps props = {};
            props.allocType = cudaMemAllocationTypePinned;
            props.location.type = cudaMemLocationTypeDevice;
            props.location.id = ctx->device;
            cudaMemPool_t made;
            CW_CUDA(cudaMemPoolCreate(&made, &props));
            uint64_t keep = ~0ull;
            CW_CUDA(cudaMemPoolSetAttribute(made, cudaMemPoolAttrReleaseThreshold, &keep));
            pools[ctx->device] = made;
        }
        pool = pools[ctx->device];
    }
    need = std::max(need, 2 * ctx->tree_scratch_bytes);
    try {
        ctx->tree_outgrown.reserve(ctx->tree_outgrown.size() + 1);
    } catch (...) {
        return set_error(CW_ERR_OOM, "cw_tree_attention: out of host memory");
    }
    void* p = nullptr;
    CW_CUDA(cudaMallocFromPoolAsync(&p, need, pool, ctx->stream));
    if (ctx->tree_scratch) ctx->tree_outgrown.push_back(ctx->tree_scratch);
    ctx->tree_scratch = p;
    ctx->tree_scratch_bytes = need;
    return CW_OK;
}

template <typename T, int DP, int WM, bool VEC>
static int tree_go(cw_ctx* ctx, const TreeArgs& a, int grid) {
    constexpr size_t smem = tr_smem<DP, 16 * WM>();
    static_assert(smem <= TR_SMEM_CAP, "shared memory");
    auto kern = k_tree<T, DP, WM, VEC>;
    CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    return launch_pdl(ctx, true, kern, dim3(grid), dim3(TR_THREADS), smem, a);
}
template <typename T, int DP, bool VEC>
static int tree_rows(cw_ctx* ctx, const TreeArgs& a, int grid) {
    if (a.bm == 16) return tree_go<T, DP, 1, VEC>(ctx, a, grid);
    if (a.bm == 32) return tree_go<T, DP, 2, VEC>(ctx, a, grid);
    if constexpr (DP <= 128) return tree_go<T, DP, 4, VEC>(ctx, a, grid);
    return set_error(CW_ERR_UNSUPPORTED, "cw_tree_attention: %d rows of %d", a.bm, DP);
}
template <typename T, bool VEC>
static int tree_dims(cw_ctx* ctx, const TreeArgs& a, int grid) {
    if (a.D <= 64) return tree_rows<T, 64, VEC>(ctx, a, grid);
    if (a.D <= 128) return tree_rows<T, 128, VEC>(ctx, a, grid);
    return tree_rows<T, 256, VEC>(ctx, a, grid);
}
template <typename T> static int tree_type(cw_ctx* ctx, const TreeArgs& a, bool vec, int grid) {
    return vec ? tree_dims<T, true>(ctx, a, grid) : tree_dims<T, false>(ctx, a, grid);
}

}  // namespace cw

using namespace cw;

extern "C" int cw_tree_attention(cw_ctx* ctx, const cw_tree_attn_args* p) {
    clear_error();
    CW_CHECK(ctx && p, CW_ERR_INVALID_ARG, "cw_tree_attention: bad arguments");
    CW_CHECK(p->type == CW_GGUF_F32 || p->type == CW_GGUF_F16 || p->type == CW_GGUF_BF16,
             CW_ERR_UNSUPPORTED, "cw_tree_attention: type %u (f32, f16 or bf16)", p->type);
    CW_CHECK(p->n_heads > 0 && p->n_kv > 0 && p->n_heads % p->n_kv == 0 && p->n_heads <= 4096,
             CW_ERR_INVALID_ARG, "cw_tree_attention: n_heads=%u n_kv=%u (need n_kv | n_heads)",
             p->n_heads, p->n_kv);
    CW_CHECK(p->head_dim > 0 && p->head_dim <= 256, CW_ERR_INVALID_ARG,
             "cw_tree_attention: head_dim %u (1..256)", p->head_dim);
    CW_CHECK(p->max_nodes > 0 && p->max_nodes <= TR_NODES, CW_ERR_INVALID_ARG,
             "cw_tree_attention: max_nodes %u (1..%d)", p->max_nodes, TR_NODES);
    CW_CHECK(p->n_req > 0 && p->n_req < (1u << 24) && p->n_rows > 0 && p->n_rows < (1u << 31),
             CW_ERR_INVALID_ARG, "cw_tree_attention: bad shape");
    CW_CHECK(p->page_size > 0 && p->page_size <= (1u << 20) && p->n_pages > 0 &&
                 p->n_pages < (1u << 31) && p->max_pages > 0 &&
                 (uint64_t)p->max_pages * p->page_size < (1ull << 31) - 2 * TR_TILE &&
                 (uint64_t)p->n_pages * p->page_size < (1ull << 40),
             CW_ERR_INVALID_ARG, "cw_tree_attention: bad cache shape");
    CW_CHECK(p->q_off < (1ull << 40) && p->q_stride < (1ull << 30) &&
                 (p->q_stride >= (uint64_t)p->n_heads * p->head_dim || p->n_rows == 1),
             CW_ERR_INVALID_ARG, "cw_tree_attention: bad q offset or stride");
    CW_CHECK(p->scale >= 0.f && std::isfinite(p->scale) && p->softcap >= 0.f &&
                 std::isfinite(p->softcap) && p->window < (1u << 31),
             CW_ERR_INVALID_ARG, "cw_tree_attention: bad scale, softcap or window");
    const size_t es = p->type == CW_GGUF_F32 ? 4 : 2, rows = p->n_rows, D = p->head_dim;
    const size_t w = p->n_heads * D, words = (p->max_nodes + 31) / 32;
    const size_t cache = (size_t)p->n_pages * p->page_size * p->n_kv * D * es;
    BufEntry *q, *k, *v, *table, *lens, *starts, *mask = nullptr, *pos = nullptr, *out;
    CW_TRY(buf_get(ctx, p->q, &q, (p->q_off + (rows - 1) * p->q_stride + w) * es,
                   "cw_tree_attention(q)"));
    CW_TRY(buf_get(ctx, p->k_cache, &k, cache, "cw_tree_attention(k_cache)"));
    CW_TRY(buf_get(ctx, p->v_cache, &v, cache, "cw_tree_attention(v_cache)"));
    CW_TRY(buf_get(ctx, p->table, &table, (size_t)p->n_req * p->max_pages * 4,
                   "cw_tree_attention(table)"));
    CW_TRY(buf_get(ctx, p->lens, &lens, (size_t)p->n_req * 4, "cw_tree_attention(lens)"));
    CW_TRY(buf_get(ctx, p->starts, &starts, ((size_t)p->n_req + 1) * 4,
                   "cw_tree_attention(starts)"));
    if (p->mask) CW_TRY(buf_get(ctx, p->mask, &mask, rows * words * 4, "cw_tree_attention(mask)"));
    if (p->window)
        CW_TRY(buf_get(ctx, p->positions, &pos, rows * 4, "cw_tree_attention(positions)"));
    CW_TRY(buf_get(ctx, p->out, &out, rows * w * es, "cw_tree_attention(out)"));
    cudaSetDevice(ctx->device);
    TreeArgs a{};
    a.q = (const char*)q->ptr + p->q_off * es;
    a.k = k->ptr;
    a.v = v->ptr;
    a.out = out->ptr;
    a.table = (const int*)table->ptr;
    a.lens = (const int*)lens->ptr;
    a.starts = (const int*)starts->ptr;
    a.mask = mask ? (const uint32_t*)mask->ptr : nullptr;
    a.positions = pos ? (const int*)pos->ptr : nullptr;
    a.q_stride = (long long)p->q_stride;
    a.n_req = (int)p->n_req;
    a.n_rows = (int)rows;
    a.max_nodes = (int)p->max_nodes;
    a.words = (int)words;
    a.H = (int)p->n_heads;
    a.K = (int)p->n_kv;
    a.G = a.H / a.K;
    a.D = (int)D;
    a.page = (int)p->page_size;
    a.n_pages = (int)p->n_pages;
    a.max_pages = (int)p->max_pages;
    a.window = (int)p->window;
    a.scale = p->scale > 0.f ? p->scale : powf((float)D, -0.5f);
    a.softcap = p->softcap;
    a.status = ctx->d_status;
    const long long most = (long long)p->max_nodes * a.G;  // rows of a request's kv head
    const bool tc = tree_tc_takes(*p, a.q, a.k, a.v);
    int grid;
    if (tc) {
        a.bm = tree_tc_rows(a);
        grid = tree_tc_grid(ctx, a);
        // an item's start and end take 2 us (64 dims, 0.41 us a tile) to 5 us (0.67 us)
        a.pad = D <= 64 ? 5 : 8;
    } else {
        a.pad = 1;
        a.bm = most <= 16 ? 16 : most <= 32 || D > 128 ? 32 : 64;
        grid = ctx->sm_count;
    }
    a.dp = (a.D + 3) / 4 * 4;
    const size_t part = (size_t)grid * 2 * a.bm * a.dp * 4, ml = (size_t)grid * 2 * a.bm * 8;
    const size_t need = part + ml + (size_t)grid * sizeof(TreePiece);
    CW_TRY(tree_scratch(ctx, need));
    a.part = (float*)ctx->tree_scratch;
    a.ml = (float2*)((char*)ctx->tree_scratch + part);
    a.pieces = (TreePiece*)((char*)ctx->tree_scratch + part + ml);
    OpScope scope(ctx, "tree_attention");
    if (tc) {
        CW_TRY(tree_tc_launch(ctx, a, p->type, grid));
    } else {
        const uint64_t every = D | (p->q_off | p->q_stride);
        const bool vec = every % 4 == 0;
        if (p->type == CW_GGUF_F32) CW_TRY(tree_type<float>(ctx, a, vec, grid));
        else if (p->type == CW_GGUF_F16) CW_TRY(tree_type<__half>(ctx, a, vec, grid));
        else CW_TRY(tree_type<__nv_bfloat16>(ctx, a, vec, grid));
    }
    const dim3 join(grid, (unsigned)((std::min<long long>(most, a.bm) + TJ_WARPS - 1) / TJ_WARPS),
                    (unsigned)((a.D + 127) / 128));
    auto jk = p->type == CW_GGUF_F32   ? k_tree_join<float>
              : p->type == CW_GGUF_F16 ? k_tree_join<__half>
                                       : k_tree_join<__nv_bfloat16>;
    CW_TRY(launch_pdl(ctx, true, jk, join, dim3(TJ_WARPS * 32), 0, a));
    return check_launch("tree_attention");
}
