// cw_norm_rope.cu -- norms of the q and k heads, their rotary positions and the append to
// a paged cache in one pass (cw_norm_rope).
//
//   n = x r w,  r = (mean(x^2) + eps)^-1/2;   y = R(position) n
//
// Memory bound: every row is read and written once.  A head row is held by L neighbouring
// lanes, C chunks of two 16-byte vectors each, placed so that a lane holds whole pairs;
// the sum of squares is added over the L lanes by shuffles.  A lane keeps its pairs' sines
// and its weights in registers and walks a share of its token's q, then k, then v heads.
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "cw_common.h"
#include "cw_rotary.cuh"

namespace cw {

struct NormRopeArgs {
    const unsigned long long* steps;
    const int *positions, *slots;
    const void *q, *k, *v;
    const float *q_norm, *k_norm;
    void *q_out, *k_out, *k_cache, *v_cache;
    long long q_stride, k_stride, v_stride;
    float amp, eps;
    int unit, rot, n_tokens, H, K, D, page;
    long long n_slots;
    int heads, lanes, groups, per;  // heads a token has; lanes of a head row; head groups; heads each
    int* status;
};

constexpr int NR_THREADS = 256;
// A head's loads are in flight while the one before is worked on, three blocks to an SM and
// at most 12 heads to a lane: 32768 bf16 rows of 32 + 8 + 8 heads in 168 us (872 MB, 5.2
// TB/s); 16384 f32 rows of 16 + 8 + 8 heads with k rows besides in 108 us (5.6 TB/s), 4096 in
// 31, 128 in 4.2.  The choices were made on the bf16 rows where this form took 163 us: 168
// before results were converted two at a time, 175 with two heads in flight, 191 with four
// blocks an SM (64 registers), 166 with 24 heads to a lane and 189 with 64, 166 with
// streaming stores, the arithmetic in paired f32 instructions no different.
constexpr int NR_PER = 12;

// Two neighbours at once: one conversion instruction for 16-bit types.
__device__ __forceinline__ void nr_set2(float* d, float x, float y) { d[0] = x, d[1] = y; }
__device__ __forceinline__ void nr_set2(__half* d, float x, float y) {
    *(__half2*)d = __floats2half2_rn(x, y);
}
__device__ __forceinline__ void nr_set2(__nv_bfloat16* d, float x, float y) {
    *(__nv_bfloat162*)d = __floats2bfloat162_rn(x, y);
}

// ALL: every lane's chunks are whole (L * C chunks of 2 * VEC elements make a head row).
template <typename T, int VEC, int C, bool HALF, bool ALL>
__global__ void __launch_bounds__(NR_THREADS, C == 1 ? 3 : 1)
    k_norm_rope(const __grid_constant__ NormRopeArgs a) {
    typedef typename VecOf<VEC * sizeof(T)>::type V;
    union alignas(16) Row {
        V v[2 * C];
        T e[2 * VEC * C];
    };
    const int L = a.lanes, sub = threadIdx.x & (L - 1);
    // (whole 32-bit numbers: 64-bit divisions took a microsecond of a small call)
    const unsigned row = blockIdx.x * (unsigned)(NR_THREADS / L) + threadIdx.x / L;
    const unsigned at = row / (unsigned)a.groups;
    // every lane stays for the shuffles: one past the last token does its work unseen
    const bool live = at < (unsigned)a.n_tokens;
    const int t = live ? (int)at : a.n_tokens - 1, g = (int)(row - at * a.groups);
    const int rot_chunks = a.rot / (2 * VEC);
    // the lane's chunks: vectors at e0 and e1, a pair's elements in different vectors (HALF)
    // or side by side; past the rotated part plain neighbours
    int e0[C], e1[C];
    bool turn[C];
#pragma unroll
    for (int i = 0; i < C; i++) {
        const int c = sub + i * L;
        turn[i] = c < rot_chunks;
        e0[i] = turn[i] ? (HALF ? c * VEC : 2 * c * VEC) : a.rot + 2 * (c - rot_chunks) * VEC;
        e1[i] = turn[i] && HALF ? e0[i] + a.rot / 2 : e0[i] + VEC;
    }
    pdl_wait();
    pdl_trigger();
    const long long pos = a.positions[t];
    long long slot = -1, dst0 = 0;
    if (a.slots) {
        slot = a.slots[t];
        if (slot >= a.n_slots) {
            if (live && sub == 0 && g == 0) atomicCAS(a.status, DEV_OK, DEV_BAD_INPUT);
            slot = -1;
        }
        if (slot >= 0) {
            const int pg = (int)slot / a.page;
            dst0 = ((long long)pg * a.K * a.page + ((int)slot - pg * a.page)) * a.D;
        }
    }
    const T* q = (const T*)a.q + t * a.q_stride;
    const T* k = (const T*)a.k + t * a.k_stride;
    const T* v = (const T*)a.v + t * a.v_stride;
    auto load = [&](int i, Row& w) {  // the lane's i-th head
        const int h = g + i * a.groups;
        if (i >= a.per || h >= a.heads || !live) return;
        const T* src = h < a.H         ? q + h * a.D
                       : h < a.H + a.K ? k + (h - a.H) * a.D
                                       : v + (h - a.H - a.K) * a.D;
#pragma unroll
        for (int j = 0; j < C; j++) {
            if (ALL || e0[j] < a.D) w.v[2 * j] = *(const V*)(src + e0[j]);
            if (ALL || e1[j] < a.D) w.v[2 * j + 1] = *(const V*)(src + e1[j]);
        }
    };
    Row w;
#pragma unroll
    for (int i = 0; i < 2 * VEC * C; i++) rp_set(&w.e[i], 0.f);
    load(0, w);
    float cs[C * VEC], sn[C * VEC];
#pragma unroll
    for (int j = 0; j < C; j++)
        if (turn[j]) rotary_sines<T, VEC>(a.steps + (sub + j * L) * VEC, pos, a.amp, cs + j * VEC, sn + j * VEC);
    float gain[2 * VEC * C];
    const float* held = nullptr;  // the weights in `gain`; without any, ones
    const float unit = a.unit ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < 2 * VEC * C; i++) gain[i] = 1.f;
    for (int i = 0; i < a.per; i++) {
        const int h = g + i * a.groups;
        Row y = w;
        load(i + 1, w);  // in flight while this head is worked on
        // the same for all lanes of a group: every lane of the warp meets the shuffles
        const bool on = h < a.heads;
        const bool norm = on && h < a.H + a.K && (h < a.H ? a.q_norm : a.k_norm);
        float r = 1.f;
        if (__any_sync(FULL, norm)) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < C; j++)
#pragma unroll
                for (int i = 0; i < 2 * VEC; i++) {
                    const float x = rp_f32(y.e[2 * VEC * j + i]);
                    if (ALL || (i < VEC ? e0[j] : e1[j]) < a.D) s = fmaf(x, x, s);
                }
            for (int o = L >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
            // (16-bit values: the fast root is off by 2^-22)
            if (norm) r = sizeof(T) == 2 ? rsqrtf(s / (float)a.D + a.eps)
                                         : 1.f / sqrtf(s / (float)a.D + a.eps);
        }
        if (!on || !live) continue;
        if (h < a.H + a.K) {
            const float* want = h < a.H ? a.q_norm : a.k_norm;
            if (want != held) {
                held = want;
#pragma unroll
                for (int j = 0; j < C; j++)
#pragma unroll
                    for (int i = 0; i < 2 * VEC; i++) {
                        const int e = i < VEC ? e0[j] + i : e1[j] + i - VEC;
                        gain[2 * VEC * j + i] = want && (ALL || e < a.D) ? want[e] + unit : 1.f;
                    }
            }
#pragma unroll
            for (int j = 0; j < C; j++) {
                float x[2 * VEC];
#pragma unroll
                for (int i = 0; i < 2 * VEC; i++)
                    x[i] = rp_f32(y.e[2 * VEC * j + i]) * r * gain[2 * VEC * j + i];
                if (turn[j]) {
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        const int p0 = HALF ? i : 2 * i, p1 = HALF ? VEC + i : 2 * i + 1;
                        const float c = cs[j * VEC + i], s = sn[j * VEC + i];
                        const float x0 = x[p0], x1 = x[p1];
                        x[p0] = x0 * c - x1 * s;
                        x[p1] = x1 * c + x0 * s;
                    }
                }
#pragma unroll
                for (int i = 0; i < 2 * VEC; i += 2)
                    nr_set2(&y.e[2 * VEC * j + i], x[i], x[i + 1]);
            }
        }
        auto put = [&](T* dst) {
#pragma unroll
            for (int j = 0; j < C; j++) {
                if (ALL || e0[j] < a.D) *(V*)(dst + e0[j]) = y.v[2 * j];
                if (ALL || e1[j] < a.D) *(V*)(dst + e1[j]) = y.v[2 * j + 1];
            }
        };
        if (h < a.H) {
            put((T*)a.q_out + ((long long)t * a.H + h) * a.D);
        } else if (h < a.H + a.K) {
            if (a.k_out) put((T*)a.k_out + ((long long)t * a.K + h - a.H) * a.D);
            if (slot >= 0)
                put((T*)a.k_cache + dst0 + (long long)(h - a.H) * a.page * a.D);
        } else if (slot >= 0) {
            put((T*)a.v_cache + dst0 + (long long)(h - a.H - a.K) * a.page * a.D);
        }
    }
}

template <typename T, int VEC, int C>
static int norm_rope_go(cw_ctx* ctx, NormRopeArgs& a, bool half, int chunks) {
    a.lanes = 1;
    while (a.lanes * C < chunks) a.lanes *= 2;
    // as many heads to a lane as leave 2048 threads an SM (768 of them are resident at a time,
    // so 2.7 waves): 1003 f16 rows of 8 + 4 + 4 heads of 256 run with one head to a lane, 2.3 waves
    const long long all = (long long)a.n_tokens * a.lanes * a.heads;
    const long long wave = (long long)ctx->sm_count * 2048;
    a.per = (int)std::max<long long>(1, std::min<long long>(all / wave, std::min(a.heads, NR_PER)));
    a.groups = (a.heads + a.per - 1) / a.per;
    const unsigned long long n = (unsigned long long)a.n_tokens * a.lanes * a.groups;
    const unsigned long long blocks = (n + NR_THREADS - 1) / NR_THREADS;
    CW_CHECK(blocks < (1ull << 31) && (unsigned long long)a.n_tokens * a.groups < (1ull << 32) - 512,
             CW_ERR_UNSUPPORTED, "cw_norm_rope: too many rows");
    // (vectors narrower than 16 bytes, and several chunks to a lane, are rare: checked only)
    constexpr bool CAN = C == 1 && VEC * sizeof(T) == 16;
    auto kern = half ? k_norm_rope<T, VEC, C, true, false> : k_norm_rope<T, VEC, C, false, false>;
    if (CAN && a.D == a.lanes * C * 2 * VEC && a.rot % (2 * VEC) == 0)
        kern = half ? k_norm_rope<T, VEC, C, true, CAN> : k_norm_rope<T, VEC, C, false, CAN>;
    CW_TRY(launch_pdl(ctx, true, kern, dim3((unsigned)blocks), dim3(NR_THREADS), 0, a));
    return check_launch("norm_rope");
}
// A head row in 32 lanes or fewer: one chunk each, or for long rows of narrow vectors several.
template <typename T, int VEC>
static int norm_rope_launch(cw_ctx* ctx, NormRopeArgs& a, bool half) {
    const int chunks = (a.D + 2 * VEC - 1) / (2 * VEC);
    if (chunks <= 32) return norm_rope_go<T, VEC, 1>(ctx, a, half, chunks);
    return norm_rope_go<T, VEC, 16 / VEC>(ctx, a, half, chunks);
}

}  // namespace cw

using namespace cw;

extern "C" int cw_norm_rope(cw_ctx* ctx, const cw_norm_rope_args* p) {
    clear_error();
    CW_CHECK(ctx && p, CW_ERR_INVALID_ARG, "cw_norm_rope: bad arguments");
    CW_CHECK(p->type == CW_GGUF_F32 || p->type == CW_GGUF_F16 || p->type == CW_GGUF_BF16,
             CW_ERR_UNSUPPORTED, "cw_norm_rope: type %u (f32, f16 or bf16)", p->type);
    CW_CHECK(p->layout <= CW_ROPE_INTERLEAVED, CW_ERR_INVALID_ARG, "cw_norm_rope: layout %u",
             p->layout);
    CW_CHECK(p->norm_kind <= 1, CW_ERR_INVALID_ARG, "cw_norm_rope: norm_kind %u", p->norm_kind);
    CW_CHECK(p->eps >= 0.f && isfinite(p->eps), CW_ERR_INVALID_ARG,
             "cw_norm_rope: eps must be finite and not negative");
    CW_CHECK(p->n_tokens > 0 && p->n_tokens < (1u << 31) && p->n_heads <= 4096 &&
                 p->n_kv <= 4096 && p->n_heads + p->n_kv > 0 && p->head_dim > 0 &&
                 p->head_dim <= 1024,
             CW_ERR_INVALID_ARG, "cw_norm_rope: bad shape");
    const size_t es = p->type == CW_GGUF_F32 ? 4 : 2, T = p->n_tokens, D = p->head_dim;
    const uint64_t big = 1ull << 40;  // keeps the byte counts below from overflowing
    CW_CHECK(p->q_off < big && p->k_off < big && p->v_off < big && p->q_stride < (1ull << 30) &&
                 p->k_stride < (1ull << 30) && p->v_stride < (1ull << 30),
             CW_ERR_INVALID_ARG, "cw_norm_rope: bad offset or stride");
    BufEntry *plan, *pos, *e = nullptr;
    CW_TRY(buf_get(ctx, p->plan, &plan, 0, "cw_norm_rope(plan)"));
    CW_CHECK(plan->rope_dim, CW_ERR_INVALID_ARG, "cw_norm_rope: not a plan of cw_rope_plan");
    CW_CHECK(plan->rope_dim <= D, CW_ERR_INVALID_ARG,
             "cw_norm_rope: the plan rotates %u of %zu elements", plan->rope_dim, D);
    CW_TRY(buf_get(ctx, p->positions, &pos, T * 4, "cw_norm_rope(positions)"));
    // what is read and what is written: an output may lie on its own input only, whose heads
    // the lanes that write them have read; another input at the same place is read by others
    struct Span {
        const char* at;
        size_t n;
        const char* what;
        int may;  // which input it may be, or -1
    } in[8], out[4];
    int ins = 0, outs = 0;
    in[ins++] = {(const char*)plan->ptr, plan->rope_dim / 2 * 8, "plan", -1};
    in[ins++] = {(const char*)pos->ptr, T * 4, "positions", -1};
    NormRopeArgs a{};
    auto norm = [&](cw_buf b, const float** to, const char* what) -> int {
        if (!b) return CW_OK;
        CW_TRY(buf_get(ctx, b, &e, D * 4, what));
        *to = (const float*)e->ptr;
        in[ins++] = {(const char*)e->ptr, D * 4, what, -1};
        return CW_OK;
    };
    // rows of w elements; contiguous ones may be written in place
    auto rows = [&](cw_buf b, uint64_t off, uint64_t stride, size_t w, const void** to,
                    const char* what) -> int {
        CW_CHECK(stride >= w || T == 1, CW_ERR_INVALID_ARG, "%s: a stride of %llu", what,
                 (unsigned long long)stride);
        CW_TRY(buf_get(ctx, b, &e, (off + (T - 1) * stride + w) * es, what));
        *to = (const char*)e->ptr + off * es;
        in[ins++] = {(const char*)*to, ((T - 1) * stride + w) * es, what, -1};
        return CW_OK;
    };
    auto result = [&](cw_buf b, size_t n, void** to, const char* what, int may) -> int {
        CW_TRY(buf_get(ctx, b, &e, n, what));
        *to = e->ptr;
        out[outs++] = {(const char*)e->ptr, n, what, may};
        return CW_OK;
    };
    const bool cache = p->n_kv && p->slots;
    if (p->n_heads) {
        const size_t w = p->n_heads * D;
        const int own = p->q_stride == w || T == 1 ? ins : -1;
        CW_TRY(rows(p->q, p->q_off, p->q_stride, w, &a.q, "cw_norm_rope(q)"));
        CW_TRY(norm(p->q_norm, &a.q_norm, "cw_norm_rope(q_norm)"));
        CW_TRY(result(p->q_out, T * w * es, &a.q_out, "cw_norm_rope(q_out)", own));
    }
    if (p->n_kv) {
        const size_t w = p->n_kv * D;
        CW_CHECK(p->k_out || cache, CW_ERR_INVALID_ARG,
                 "cw_norm_rope: k has neither k_out nor a cache to go to");
        const int own = p->k_stride == w || T == 1 ? ins : -1;
        CW_TRY(rows(p->k, p->k_off, p->k_stride, w, &a.k, "cw_norm_rope(k)"));
        CW_TRY(norm(p->k_norm, &a.k_norm, "cw_norm_rope(k_norm)"));
        if (p->k_out)
            CW_TRY(result(p->k_out, T * w * es, &a.k_out, "cw_norm_rope(k_out)", own));
        if (cache) {
            CW_CHECK(p->page_size > 0 && p->page_size <= (1u << 20) && p->n_pages > 0 &&
                         (uint64_t)p->n_pages * p->page_size < (1ull << 31),
                     CW_ERR_INVALID_ARG, "cw_norm_rope: bad cache shape");
            CW_TRY(rows(p->v, p->v_off, p->v_stride, w, &a.v, "cw_norm_rope(v)"));
            CW_TRY(buf_get(ctx, p->slots, &e, T * 4, "cw_norm_rope(slots)"));
            a.slots = (const int*)e->ptr;
            in[ins++] = {(const char*)e->ptr, T * 4, "slots", -1};
            const size_t n = (size_t)p->n_pages * p->page_size * w * es;
            CW_TRY(result(p->k_cache, n, &a.k_cache, "cw_norm_rope(k_cache)", -1));
            CW_TRY(result(p->v_cache, n, &a.v_cache, "cw_norm_rope(v_cache)", -1));
            a.page = (int)p->page_size;
            a.n_slots = (long long)p->n_pages * p->page_size;
        }
    }
    for (int o = 0; o < outs; o++) {
        for (int i = 0; i < ins; i++)
            CW_CHECK((i == out[o].may && out[o].at == in[i].at) ||
                         !spans_meet(out[o].at, out[o].n, in[i].at, in[i].n),
                     CW_ERR_INVALID_ARG, "%s lies on %s", out[o].what, in[i].what);
        for (int i = 0; i < o; i++)
            CW_CHECK(!spans_meet(out[o].at, out[o].n, out[i].at, out[i].n), CW_ERR_INVALID_ARG,
                     "%s lies on %s", out[o].what, out[i].what);
    }
    a.steps = (const unsigned long long*)plan->ptr;
    a.amp = plan->rope_amp;
    a.eps = p->eps;
    a.unit = (int)p->norm_kind;
    a.positions = (const int*)pos->ptr;
    a.q_stride = (long long)p->q_stride;
    a.k_stride = (long long)p->k_stride;
    a.v_stride = (long long)p->v_stride;
    a.rot = (int)plan->rope_dim;
    a.n_tokens = (int)T;
    a.H = (int)p->n_heads;
    a.K = (int)p->n_kv;
    a.D = (int)D;
    a.heads = a.H + (cache ? 2 : 1) * a.K;
    a.status = ctx->d_status;
    // the widest vector that divides the rotated halves, the rows and their places
    uint64_t every = (uint64_t)(a.rot / 2) | D;
    auto place = [&](const void* x, uint64_t stride) {  // in elements
        if (x) every |= (uint64_t)(uintptr_t)x / es | (T > 1 ? stride : 0);
    };
    place(a.q, p->q_stride);
    place(a.k, p->k_stride);
    place(a.v, p->v_stride);
    place(a.q_out, 0);
    place(a.k_out, 0);
    place(a.k_cache, 0);
    place(a.v_cache, 0);
    const uint64_t vec = std::min<uint64_t>(every & (~every + 1), 16 / es);
    cudaSetDevice(ctx->device);
    OpScope scope(ctx, "norm_rope");
    const bool half = p->layout == CW_ROPE_HALF;
    auto go = [&](auto tag) -> int {
        typedef decltype(tag) T_;
        if constexpr (sizeof(T_) == 2)
            if (vec == 8) return norm_rope_launch<T_, 8>(ctx, a, half);
        if (vec == 4) return norm_rope_launch<T_, 4>(ctx, a, half);
        if (vec == 2) return norm_rope_launch<T_, 2>(ctx, a, half);
        return norm_rope_launch<T_, 1>(ctx, a, half);
    };
    if (p->type == CW_GGUF_F32) return go(float());
    if (p->type == CW_GGUF_F16) return go(__half());
    return go(__nv_bfloat16());
}
