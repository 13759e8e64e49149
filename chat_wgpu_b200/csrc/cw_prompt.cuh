// cw_prompt.cuh -- what the kernels of cw_prompt_attention share.
//
// For one kv head a request with n rows is a block of n * G query rows (G query heads per
// kv head, row = i * G + g).  An ITEM is one kv head and up to BT rows of one request.
// Which rows those are is device data, so the grid has a SLOT for every block there can
// be: request r owns slots floor(starts[r] / BT) + r on, which is enough for its
// ceil(n / BT) blocks and ascends in r, so an item finds its request by a search and no
// sum over the requests is formed.  Slots without rows end at once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "cw_common.h"
#include "cw_device.cuh"

namespace cw {

struct PromptPiece {  // an item whose first piece is this CTA's last one
    int row0, rows, head, count, slot;
};

struct PromptArgs {
    const void *q, *k, *v;
    void* out;
    const int *starts, *key_starts;
    long long q_stride, k_stride, v_stride;
    int n_req, n_rows, n_keys, H, K, G, D, window;
    float scale, softcap;
    // f32 on the tensor cores: magnitudes of each request's kv heads, [n_req][K][PR_MAGS] (f32
    // bits; PrMag), and what the q rows were divided by, [n_rows][H]
    uint32_t* amax;
    float* q_back;
    // partial states of items that a CTA's run cuts, two to a CTA: [grid * 2][rows][dp] sums,
    // [grid * 2][rows] reference and sum of the weights (-1: no tile), and [grid] items
    float* part;
    float2* ml;
    PromptPiece* pieces;
    int cut, dp;
    int bt;     // rows of an item
    int slots;  // blocks there can be
    int* status;
};

__device__ __forceinline__ void prompt_bad(const PromptArgs& a) {
    atomicCAS(a.status, DEV_OK, DEV_BAD_INPUT);
}

struct PromptItem {
    int req;
    int row0, rows;  // its rows of q and out
    int key0, keys;  // its request's keys
    int past;        // row i of the item sees keys [.., past + i] of the request
    int first;       // first key that one of its rows may see
    int end;         // one past the last key that one of its rows may see
};

// The rows of slot s, of any kv head; rows = 0: none.
__device__ __forceinline__ PromptItem prompt_item(const PromptArgs& a, int s) {
    int lo = 0, hi = a.n_req;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const int m = min(max(a.starts[mid], 0), a.n_rows);
        if (m / a.bt + mid <= s) lo = mid;
        else hi = mid;
    }
    PromptItem it;
    const int r0 = min(max(a.starts[lo], 0), a.n_rows);
    const int r1 = min(max(a.starts[lo + 1], r0), a.n_rows);
    const int n = r1 - r0, block = s - (r0 / a.bt + lo);
    it.req = lo;
    const int* ks = a.key_starts ? a.key_starts : a.starts;
    it.key0 = min(max(ks[lo], 0), a.n_keys);
    it.keys = min(max(ks[lo + 1], it.key0), a.n_keys) - it.key0;
    const int i0 = block * a.bt;
    it.rows = block < 0 || i0 >= n ? 0 : min(a.bt, n - i0);
    it.row0 = r0 + i0;
    it.past = i0 + it.keys - n;
    it.first = a.window > 0 ? max(0, it.past - a.window + 1) : 0;
    it.end = max(0, min(it.keys, it.past + it.rows));
    return it;
}
// The CTA that meets slot 0 looks all starts over (any number of threads).
__device__ __forceinline__ void prompt_check(const PromptArgs& a, int tid, int threads) {
    bool bad = false;
    for (int r = tid; r <= a.n_req; r += threads) {
        const int s = a.starts[r], b = r ? a.starts[r - 1] : 0;
        bad |= s < b || s > a.n_rows;
        if (a.key_starts) {
            const int k = a.key_starts[r], c = r ? a.key_starts[r - 1] : 0;
            bad |= k < c || k > a.n_keys;
        } else {
            bad |= s > a.n_keys;
        }
    }
    if (bad) prompt_bad(a);
}

// Operands as pairs h + l: values are multiplied by 2^s so that the largest, `bits`, lies in
// [2^14, 2^15), and l is kept 2^11 times as large.  What is not finite, or so large that
// products could leave f32's range, is left to the f32 kernel.  So are a request and kv head
// with rows of k or v (a token's head) whose largest values are more than PR_APART powers of
// two apart: a pair loses up to 2^-50 of the largest in sight or out of it, which is then
// 2^-34 of any row's own largest, and a weight 2^-49 of the heaviest, which times any row of v
// is then below 2^-32 of the heaviest key's row.  (Rows of zeros are exact.)
constexpr uint32_t PR_ODD = (127u + 60) << 23;
constexpr uint32_t PR_APART = 16;
// 2^s is at most 2^100 (k's and q's are multiplied together), so what is smaller than this is
// left out as well, but for zeros.
constexpr uint32_t PR_TINY = (127u - 86) << 23;
// Of k and v the largest value, of q only what does not fit; of the rows of k and v the
// smallest of their largest values but 0, as its complement (the words start at 0).
enum PrMag { PR_K, PR_V, PR_Q, PR_K_LEAST, PR_V_LEAST, PR_MAGS };
__device__ __forceinline__ int pr_shift(uint32_t bits) {
    return bits ? min(14 - ((int)(bits >> 23) - 127), 100) : 0;
}
__device__ __forceinline__ bool pr_misfit(uint32_t bits) {
    return bits >= PR_ODD || (bits && bits < PR_TINY);
}
__device__ __forceinline__ bool pr_odd(const PromptArgs& a, int req, int head) {
    const uint32_t* m = a.amax + ((size_t)req * a.K + head) * PR_MAGS;
    auto apart = [](uint32_t most, uint32_t least) {  // no row but of zeros: 0 and ~0
        return most && (most >> 23) - (~least >> 23) > PR_APART;
    };
    return pr_misfit(m[PR_K]) || pr_misfit(m[PR_V]) || pr_misfit(m[PR_Q]) ||
           apart(m[PR_K], m[PR_K_LEAST]) || apart(m[PR_V], m[PR_V_LEAST]);
}

template <typename T> __device__ __forceinline__ float pr_f32(T x);
template <> __device__ __forceinline__ float pr_f32(float x) { return x; }
template <> __device__ __forceinline__ float pr_f32(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float pr_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T pr_to(float x);
template <> __device__ __forceinline__ float pr_to(float x) { return x; }
template <> __device__ __forceinline__ __half pr_to(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 pr_to(float x) { return __float2bfloat16_rn(x); }

// A row's result from its pieces, by a warp: out = sum_i w_i o_i / sum_i w_i l_i, w_i = 2^(m_i -
// max m), in key order; place(i) is piece i's row in part and ml.  A lane holds a piece's
// weight, then four dims (eight past 128) of every piece.  Bound by its dependent reads.
template <typename T, typename F>
__device__ __forceinline__ void prompt_join_row(const PromptArgs& a, int count, T* out, F piece) {
    const int lane = threadIdx.x & 31;
    float top = -INFINITY, l = 0.f;
    for (int i = lane; i < count; i += 32) {
        const float2 x = a.ml[piece(i)];
        if (!(x.y < 0.f)) top = fmaxf(top, x.x);
    }
    top = warp_max(top);
    float4 o[2] = {};
    for (int i0 = 0; i0 < count; i0 += 32) {
        float w = 0.f;
        bool live = false;  // had a tile: a piece without weight keeps the NaN of its values
        if (i0 + lane < count) {
            const float2 x = a.ml[piece(i0 + lane)];
            live = !(x.y < 0.f);
            if (live && x.x != -INFINITY) w = exp2f(x.x - top);
            if (live && x.y != 0.f) l += x.y * w;
        }
        const unsigned on = __ballot_sync(FULL, live);
        const int n = min(32, count - i0);
#pragma unroll 4
        for (int i = 0; i < n; i++) {
            const float wi = __shfl_sync(FULL, w, i);
            if (!(on >> i & 1)) continue;
            const float* from = a.part + piece(i0 + i) * a.dp;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int d = h * 128 + lane * 4;
                if (d >= a.dp) continue;
                const float4 x = *(const float4*)(from + d);
                o[h].x = fmaf(wi, x.x, o[h].x);
                o[h].y = fmaf(wi, x.y, o[h].y);
                o[h].z = fmaf(wi, x.z, o[h].z);
                o[h].w = fmaf(wi, x.w, o[h].w);
            }
        }
    }
    l = warp_sum(l);
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const float y[4] = {o[h].x, o[h].y, o[h].z, o[h].w};
        const int d = h * 128 + lane * 4;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (d + e < a.D) out[d + e] = pr_to<T>(inv == 0.f ? 0.f : y[e] * inv);
    }
}

// cw_prompt_tc.cu: on the tcgen05 tensor cores, where the shape allows it.  For f32 the
// items that pr_odd leaves out are the caller's (a.amax and a.q_back are set).
bool prompt_tc_takes(const PromptArgs& a, uint32_t type);
int prompt_tc_launch(cw_ctx* ctx, PromptArgs& a, uint32_t type);

}  // namespace cw
