// cw_paged.cu -- the page plan of a step over a paged cache (cw_page_plan) and
// the rotary positions that write to it (cw_rope_plan, cw_rope_append).
#include <cuda_bf16.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <vector>

#include "cw_common.h"
#include "cw_device.cuh"

namespace cw {

// ---- page plan -----------------------------------------------------------------
// Two exclusive sums over the requests decide everything: tokens (starts) and
// fresh pages (first).  Every CTA forms both over all requests in its shared
// memory (8 bytes per request, read from L2) and then fills its own share of the
// rows and of the fresh pages, so the plan is one launch with no word passed
// between CTAs.  Rows whose page existed read the table below `have`, rows on
// fresh pages read the free list itself: no CTA reads what another writes.  8 requests
// take 5 us (launch and dependent reads), 1500 requests with a million tokens 10 us,
// whose 13 MB alone would take 2.
constexpr int PP_THREADS = 512;
constexpr int PP_MAX_REQ = 16384;  // 3 * 4 bytes each: 192 KB of shared memory

struct PagePlanArgs {
    const int *lens, *news, *free_pages, *depths;
    int *table, *starts, *positions, *slots, *owners, *used;
    int n_req, page, shift, max_pages, n_free, max_tokens;  // shift: page = 1 << shift, or -1
};

__device__ __forceinline__ int pp_div(const PagePlanArgs& a, int x) {
    return a.shift >= 0 ? x >> a.shift : x / a.page;
}
__device__ __forceinline__ int pp_pages(const PagePlanArgs& a, long long tokens) {
    const long long p = tokens < INT_MAX - a.page ? pp_div(a, (int)tokens + a.page - 1)
                                                  : (tokens + a.page - 1) / a.page;
    return (int)min(p, (long long)a.max_pages);
}

// The last i in [0, n) with a[i] <= x (a ascending, a[0] = 0 <= x).
__device__ __forceinline__ int pp_find(const int* a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PP_THREADS) k_page_plan(PagePlanArgs a) {
    extern __shared__ int pp_sm[];
    int* s_start = pp_sm;              // [n_req] tokens before the request
    int* s_first = pp_sm + a.n_req;    // [n_req] fresh pages before it
    int* s_len = s_first + a.n_req;    // [n_req] cached tokens
    __shared__ long long w_tok[PP_THREADS / 32];
    __shared__ int w_pg[PP_THREADS / 32];
    __shared__ long long s_tokens;
    __shared__ int s_pages;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = a.n_req;
    pdl_wait();
    for (int r = tid; r < R; r += PP_THREADS) {
        const int c = max(a.lens[r], 0), n = max(a.news[r], 0);
        s_start[r] = n;
        s_first[r] = pp_pages(a, (long long)c + n) - pp_pages(a, c);
        s_len[r] = c;
    }
    __syncthreads();
    // each thread sums a run of requests, then the runs are scanned
    const int run = (R + PP_THREADS - 1) / PP_THREADS;
    const int r0 = min(tid * run, R), r1 = min(r0 + run, R);
    long long tok = 0;
    int pg = 0;
    for (int r = r0; r < r1; r++) {
        tok += s_start[r];
        pg += s_first[r];
    }
    long long itok = tok;
    int ipg = pg;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(FULL, itok, o);
        const int y = __shfl_up_sync(FULL, ipg, o);
        if (lane >= o) {
            itok += x;
            ipg += y;
        }
    }
    if (lane == 31) {
        w_tok[warp] = itok;
        w_pg[warp] = ipg;
    }
    __syncthreads();
    long long btok = itok - tok;
    int bpg = ipg - pg;
#pragma unroll
    for (int w = 0; w < PP_THREADS / 32; w++)
        if (w < warp) {
            btok += w_tok[w];
            bpg += w_pg[w];
        }
    for (int r = r0; r < r1; r++) {
        const int n = s_start[r], f = s_first[r];
        s_start[r] = (int)min(btok, (long long)INT_MAX);
        s_first[r] = bpg;
        btok += n;
        bpg += f;
    }
    if (tid == PP_THREADS - 1) {  // the last run ends at R (empty runs carry the sum)
        s_tokens = btok;
        s_pages = bpg;
    }
    __syncthreads();
    const int tokens = (int)min(s_tokens, (long long)INT_MAX), pages = s_pages;
    if (blockIdx.x == 0) {
        for (int r = tid; r < R; r += PP_THREADS) a.starts[r] = s_start[r];
        if (tid == 0) {
            a.starts[R] = tokens;
            a.used[0] = pages;
        }
    }
    const int step = gridDim.x * PP_THREADS, g0 = blockIdx.x * PP_THREADS + tid;
    // fresh pages into the table, -1 for those that lack: what an earlier step left there
    // may be another request's page by now
    for (int u = g0; u < pages; u += step) {
        const int r = pp_find(s_first, R, u);  // the last request starting at or before u
        const int have = pp_pages(a, s_len[r]);
        a.table[(size_t)r * a.max_pages + have + (u - s_first[r])] =
            u < a.n_free ? a.free_pages[u] : -1;
    }
    // token rows, four to a thread (16-byte stores)
    const int groups = (a.max_tokens + 3) / 4;
    for (int g = g0; g < groups; g += step) {
        const int t0 = g * 4;
        int pos[4], slot[4], own[4];
        int r = t0 < tokens ? pp_find(s_start, R, t0) : 0;
        int c = 0, have = 0, first = 0, begin = 0, end = -1, page_at = -1, page_id = -1;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = t0 + i;
            pos[i] = 0;
            slot[i] = own[i] = -1;
            if (t >= tokens || t >= a.max_tokens) continue;
            if (t >= end) {  // into request r, past empty ones
                if (end >= 0) r++;
                while (r + 1 < R && s_start[r + 1] <= t) r++;
                begin = s_start[r];
                end = r + 1 < R ? s_start[r + 1] : tokens;
                c = s_len[r];
                have = pp_pages(a, c);
                first = s_first[r];
                page_at = -1;
            }
            const long long at = (long long)c + (t - begin);
            const int ap = at < INT_MAX ? pp_div(a, (int)at) : INT_MAX;
            if (ap != page_at) {
                page_at = ap;
                page_id = -1;
                if (ap < have) {
                    page_id = a.table[(size_t)r * a.max_pages + ap];
                } else if (ap < a.max_pages) {
                    const int u = first + ap - have;
                    if (u < a.n_free) page_id = a.free_pages[u];
                }
            }
            pos[i] = a.depths ? c + a.depths[t] : (int)at;
            own[i] = r;
            if (page_id >= 0)  // past 31 bits: a slot that no cache has
                slot[i] = (int)min((long long)page_id * a.page + ((int)at - ap * a.page),
                                   (long long)INT_MAX);
        }
        if (t0 + 4 <= a.max_tokens) {
            ((int4*)a.positions)[g] = make_int4(pos[0], pos[1], pos[2], pos[3]);
            ((int4*)a.slots)[g] = make_int4(slot[0], slot[1], slot[2], slot[3]);
            ((int4*)a.owners)[g] = make_int4(own[0], own[1], own[2], own[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (t0 + i < a.max_tokens) {
                    a.positions[t0 + i] = pos[i];
                    a.slots[t0 + i] = slot[i];
                    a.owners[t0 + i] = own[i];
                }
        }
    }
}

// ---- rotary positions + append ---------------------------------------------------
// y0 = x0 cos(p f) - x1 sin(p f), y1 = x1 cos(p f) + x0 sin(p f) per pair.  The
// angle p f is formed in turns as 64-bit fixed point: p * round(f/2pi * 2^64)
// wraps modulo one turn exactly, so the f32 that goes to sincospif is within half
// a turn at any position (an f32 product p * f is off by 2^-24 of the whole
// angle: 0.004 rad at position 100000).
// Memory bound: every row is read and written once.  A thread owns VEC pairs (two
// 16-byte vectors) of one token and walks a share of the token's q, k and v
// heads, so one set of sines serves all of them; neighbouring threads take
// neighbouring vectors, then neighbouring heads.  32768 bf16 rows of 32 + 8 + 8 heads
// take 142 us (805 MB, 5.7 TB/s; 8 heads to a thread took 166, 2 took 294), 4096 f32
// rows of 16 + 8 + 8 heads 27 us (4.9 TB/s).
struct RopeArgs {
    const unsigned long long* steps;
    const int *positions, *slots;
    const void *q, *k, *v;
    void *q_out, *k_cache, *v_cache;
    long long q_stride, k_stride, v_stride;
    float amp;
    int rot, n_tokens, H, K, D, page;
    long long n_slots;
    int chunks, groups, per;  // 2*VEC-element chunks of a head row; head groups; heads each
    int* status;
};

template <int BYTES> struct VecOf;
template <> struct VecOf<16> { typedef uint4 type; };
template <> struct VecOf<8> { typedef uint2 type; };
template <> struct VecOf<4> { typedef uint32_t type; };
template <> struct VecOf<2> { typedef uint16_t type; };

__device__ __forceinline__ float rp_f32(float x) { return x; }
__device__ __forceinline__ float rp_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float rp_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void rp_set(float* d, float x) { *d = x; }
__device__ __forceinline__ void rp_set(__half* d, float x) { *d = __float2half_rn(x); }
__device__ __forceinline__ void rp_set(__nv_bfloat16* d, float x) { *d = __float2bfloat16_rn(x); }

constexpr int RP_THREADS = 256;
constexpr int RP_UNROLL = 2;  // heads whose loads are in flight while two others are turned

template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(RP_THREADS, 3) k_rope_append(RopeArgs a) {
    typedef typename VecOf<VEC * sizeof(T)>::type V;
    union Row {
        V v[2];
        T e[2 * VEC];
    };
    const int per_token = a.chunks * a.groups;
    const unsigned long long base = (unsigned long long)blockIdx.x * RP_THREADS;
    const unsigned long long tb = base / per_token;
    const unsigned in = (unsigned)(base - tb * per_token) + threadIdx.x;
    const unsigned long long t64 = tb + in / per_token;
    if (t64 >= (unsigned long long)a.n_tokens) return;
    const int t = (int)t64, x = (int)(in % per_token);
    const int c = x % a.chunks, g = x / a.chunks;
    const int rot_chunks = a.rot / (2 * VEC);
    const bool turn = c < rot_chunks;
    // the chunk's two vectors: a pair's elements in different vectors (HALF) or
    // side by side; past the rotated part plain neighbours
    const int e0 = turn ? (HALF ? c * VEC : 2 * c * VEC) : a.rot + 2 * (c - rot_chunks) * VEC;
    const int e1 = turn && HALF ? e0 + a.rot / 2 : e0 + VEC;
    const bool two = e1 < a.D;
    const int heads = a.H + 2 * a.K;
    pdl_wait();
    const long long pos = a.positions[t];
    long long slot = -1, dst0 = 0;
    if (a.K) {
        slot = a.slots[t];
        if (slot >= a.n_slots) {
            if (x == 0) atomicCAS(a.status, DEV_OK, DEV_BAD_INPUT);
            slot = -1;
        }
        if (slot >= 0) {
            const long long pg = slot / a.page;
            dst0 = (pg * a.K * a.page + (slot - pg * a.page)) * a.D;
        }
    }
    const T* q = (const T*)a.q + t * a.q_stride;
    const T* k = (const T*)a.k + t * a.k_stride;
    const T* v = (const T*)a.v + t * a.v_stride;
    auto load = [&](int i, Row& w) {  // the thread's i-th head
        const int h = g + i * a.groups;
        if (i >= a.per || h >= heads) return;
        const T* src = h < a.H         ? q + h * a.D
                       : h < a.H + a.K ? k + (h - a.H) * a.D
                                       : v + (h - a.H - a.K) * a.D;
        w.v[0] = *(const V*)(src + e0);
        if (two) w.v[1] = *(const V*)(src + e1);
    };
    Row w[RP_UNROLL];
#pragma unroll
    for (int u = 0; u < RP_UNROLL; u++) load(u, w[u]);
    float cs[VEC], sn[VEC];
    if (turn) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const long long ph =
                (long long)((unsigned long long)pos * a.steps[c * VEC + i]);
            // 16-bit values: within half a turn the fast functions are off by 2^-21
            if (sizeof(T) == 2) __sincosf((float)ph * 0x1.921fb6p-62f, &sn[i], &cs[i]);
            else sincospif((float)ph * 0x1p-63f, &sn[i], &cs[i]);
            sn[i] *= a.amp;
            cs[i] *= a.amp;
        }
    }
    for (int i0 = 0; i0 < a.per; i0 += RP_UNROLL) {
#pragma unroll
        for (int u = 0; u < RP_UNROLL; u++) {
            const int h = g + (i0 + u) * a.groups;
            Row y = w[u];
            load(i0 + RP_UNROLL + u, w[u]);  // in flight while this head is turned
            if (i0 + u >= a.per || h >= heads) continue;
            T* dst;
            if (h < a.H) {
                dst = (T*)a.q_out + ((long long)t * a.H + h) * a.D;
            } else {
                if (slot < 0) continue;
                dst = h < a.H + a.K ? (T*)a.k_cache + dst0 + (long long)(h - a.H) * a.page * a.D
                                    : (T*)a.v_cache + dst0 +
                                          (long long)(h - a.H - a.K) * a.page * a.D;
            }
            if (turn && h < a.H + a.K) {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    T* p0 = HALF ? &y.e[i] : &y.e[2 * i];
                    T* p1 = HALF ? &y.e[VEC + i] : &y.e[2 * i + 1];
                    const float x0 = rp_f32(*p0), x1 = rp_f32(*p1);
                    rp_set(p0, x0 * cs[i] - x1 * sn[i]);
                    rp_set(p1, x1 * cs[i] + x0 * sn[i]);
                }
            }
            *(V*)(dst + e0) = y.v[0];
            if (two) *(V*)(dst + e1) = y.v[1];
        }
    }
}

template <typename T, int VEC>
static int rope_launch(cw_ctx* ctx, RopeArgs a, bool half) {
    const int heads = a.H + 2 * a.K;
    a.chunks = a.rot / (2 * VEC) + (a.D - a.rot + 2 * VEC - 1) / (2 * VEC);
    // as many heads to a thread as still leave one full wave of threads
    const long long all = (long long)a.n_tokens * a.chunks * heads;
    const long long wave = (long long)ctx->sm_count * 2048;
    a.per = (int)std::max<long long>(1, std::min<long long>(all / wave, heads));
    if (a.per >= RP_UNROLL) a.per = a.per / RP_UNROLL * RP_UNROLL;
    a.groups = (heads + a.per - 1) / a.per;
    const unsigned long long n = (unsigned long long)a.n_tokens * a.chunks * a.groups;
    const unsigned long long blocks = (n + RP_THREADS - 1) / RP_THREADS;
    CW_CHECK(blocks < (1ull << 31), CW_ERR_UNSUPPORTED, "cw_rope_append: too many rows");
    CW_TRY(launch_pdl(ctx, true, half ? k_rope_append<T, VEC, true> : k_rope_append<T, VEC, false>,
                      dim3((unsigned)blocks), dim3(RP_THREADS), 0, a));
    return check_launch("rope_append");
}

}  // namespace cw

using namespace cw;

extern "C" {

int cw_page_plan(cw_ctx* ctx, const cw_page_plan_args* p) {
    clear_error();
    CW_CHECK(ctx && p, CW_ERR_INVALID_ARG, "cw_page_plan: bad arguments");
    CW_CHECK(p->n_req > 0 && p->n_req <= PP_MAX_REQ, CW_ERR_INVALID_ARG,
             "cw_page_plan: n_req %u (1..%d)", p->n_req, PP_MAX_REQ);
    CW_CHECK(p->page_size > 0 && p->page_size <= (1u << 20) && p->max_pages > 0 &&
                 (uint64_t)p->n_req * p->max_pages < (1ull << 31) && p->n_free < (1u << 31) &&
                 p->max_tokens < (1u << 31) - 4,
             CW_ERR_INVALID_ARG, "cw_page_plan: bad shape");
    const size_t R = p->n_req, T = p->max_tokens;
    BufEntry *lens, *news, *fp = nullptr, *table, *depths = nullptr, *starts, *pos = nullptr,
             *slots = nullptr, *owners = nullptr, *used;
    CW_TRY(buf_get(ctx, p->lens, &lens, R * 4, "cw_page_plan(lens)"));
    CW_TRY(buf_get(ctx, p->news, &news, R * 4, "cw_page_plan(news)"));
    if (p->n_free)
        CW_TRY(buf_get(ctx, p->free_pages, &fp, (size_t)p->n_free * 4, "cw_page_plan(free_pages)"));
    CW_TRY(buf_get(ctx, p->table, &table, R * p->max_pages * 4, "cw_page_plan(table)"));
    if (p->depths) CW_TRY(buf_get(ctx, p->depths, &depths, T * 4, "cw_page_plan(depths)"));
    CW_TRY(buf_get(ctx, p->starts, &starts, (R + 1) * 4, "cw_page_plan(starts)"));
    CW_TRY(buf_get(ctx, p->used, &used, 4, "cw_page_plan(used)"));
    if (T) {
        CW_TRY(buf_get(ctx, p->positions, &pos, T * 4, "cw_page_plan(positions)"));
        CW_TRY(buf_get(ctx, p->slots, &slots, T * 4, "cw_page_plan(slots)"));
        CW_TRY(buf_get(ctx, p->owners, &owners, T * 4, "cw_page_plan(owners)"));
    }
    cudaSetDevice(ctx->device);
    PagePlanArgs a{};
    a.lens = (const int*)lens->ptr;
    a.news = (const int*)news->ptr;
    a.free_pages = fp ? (const int*)fp->ptr : nullptr;
    a.depths = depths ? (const int*)depths->ptr : nullptr;
    a.table = (int*)table->ptr;
    a.starts = (int*)starts->ptr;
    a.positions = pos ? (int*)pos->ptr : nullptr;
    a.slots = slots ? (int*)slots->ptr : nullptr;
    a.owners = owners ? (int*)owners->ptr : nullptr;
    a.used = (int*)used->ptr;
    a.n_req = (int)R;
    a.page = (int)p->page_size;
    a.max_pages = (int)p->max_pages;
    a.n_free = (int)p->n_free;
    a.max_tokens = (int)T;
    a.shift = (p->page_size & (p->page_size - 1)) == 0 ? __builtin_ctz(p->page_size) : -1;
    const size_t smem = 12 * R;
    // 48 KB without it, the kernel's own 208 bytes of static shared memory included
    if (smem > 47 * 1024)
        CW_CUDA(cudaFuncSetAttribute(k_page_plan, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     12 * PP_MAX_REQ));
    // one group of four rows to a thread until two CTAs per SM are busy
    const long long items = std::max<long long>((long long)(T + 3) / 4, 1);
    const int grid = (int)std::min<long long>((items + PP_THREADS - 1) / PP_THREADS,
                                              2ll * ctx->sm_count);
    OpScope scope(ctx, "page_plan");
    CW_TRY(launch_pdl(ctx, true, k_page_plan, dim3(grid), dim3(PP_THREADS), smem, a));
    return check_launch("page_plan");
}

int cw_rope_plan(cw_ctx* ctx, size_t rot_dim, double theta, const cw_rope_scaling* sc,
                 cw_buf* plan) {
    clear_error();
    CW_CHECK(ctx && plan, CW_ERR_INVALID_ARG, "cw_rope_plan: bad arguments");
    CW_CHECK(rot_dim >= 2 && rot_dim <= 1024 && rot_dim % 2 == 0, CW_ERR_INVALID_ARG,
             "cw_rope_plan: rot_dim %zu (even, 2..1024)", rot_dim);
    CW_CHECK(theta >= 1.0 && isfinite(theta), CW_ERR_INVALID_ARG,
             "cw_rope_plan: theta must be finite and at least 1");
    const uint32_t kind = sc ? sc->kind : CW_ROPE_PLAIN;
    CW_CHECK(kind <= CW_ROPE_YARN, CW_ERR_INVALID_ARG, "cw_rope_plan: scaling kind %u", kind);
    if (kind != CW_ROPE_PLAIN)
        CW_CHECK(sc->factor > 0 && isfinite(sc->factor), CW_ERR_INVALID_ARG,
                 "cw_rope_plan: factor must be positive");
    if (kind >= CW_ROPE_BANDED)
        CW_CHECK(sc->trained > 0 && sc->low > 0 && sc->high > sc->low && isfinite(sc->high) &&
                     (kind != CW_ROPE_YARN || theta > 1.0) && isfinite(sc->amplitude),
                 CW_ERR_INVALID_ARG, "cw_rope_plan: needs trained > 0 and 0 < low < high");
    const double two_pi = 6.283185307179586476925286766559;
    double amp = 1.0, lo = 0.0, hi = 0.0;
    if (kind == CW_ROPE_YARN) {
        // the (fractional) pair index that makes `turns` turns within `trained`
        auto at = [&](double turns) {
            return (double)rot_dim * log((double)sc->trained / (turns * two_pi)) /
                   (2.0 * log(theta));
        };
        lo = std::max(floor(at(sc->high)), 0.0);
        hi = std::min(ceil(at(sc->low)), (double)rot_dim - 1.0);
        amp = sc->amplitude != 0.f ? (double)sc->amplitude : 0.1 * log((double)sc->factor) + 1.0;
    }
    try {
        std::vector<uint64_t> steps(rot_dim / 2);
        for (size_t i = 0; i < steps.size(); i++) {
            double f = pow(theta, -2.0 * (double)i / (double)rot_dim);
            if (kind == CW_ROPE_LINEAR) {
                f /= sc->factor;
            } else if (kind == CW_ROPE_BANDED) {
                const double turns = sc->trained * f / two_pi;
                const double keep = std::min(
                    std::max((turns - sc->low) / ((double)sc->high - sc->low), 0.0), 1.0);
                f = f / sc->factor * (1.0 - keep) + f * keep;
            } else if (kind == CW_ROPE_YARN) {
                const double ramp =
                    std::min(std::max(((double)i - lo) / std::max(hi - lo, 1e-3), 0.0), 1.0);
                f = f / sc->factor * ramp + f * (1.0 - ramp);
            }
            const double turns = fmod(f / two_pi, 1.0);  // whole turns drop out
            steps[i] = (uint64_t)nearbyint(ldexp(turns, 64));
        }
        cudaSetDevice(ctx->device);
        BufEntry* e;
        cw_buf b;
        CW_TRY(buf_new(ctx, steps.size() * 8, BUF_PERSISTENT, &b, &e));
        e->rope_dim = (uint32_t)rot_dim;
        e->rope_amp = (float)amp;
        CW_CUDA(cudaMemcpyAsync(e->ptr, steps.data(), steps.size() * 8, cudaMemcpyHostToDevice,
                                ctx->stream));
        CW_CUDA(cudaStreamSynchronize(ctx->stream));  // before `steps` goes
        *plan = b;
    } catch (...) {
        return set_error(CW_ERR_OOM, "cw_rope_plan: out of host memory");
    }
    return CW_OK;
}

int cw_rope_append(cw_ctx* ctx, const cw_rope_append_args* p) {
    clear_error();
    CW_CHECK(ctx && p, CW_ERR_INVALID_ARG, "cw_rope_append: bad arguments");
    CW_CHECK(p->type == CW_GGUF_F32 || p->type == CW_GGUF_F16 || p->type == CW_GGUF_BF16,
             CW_ERR_UNSUPPORTED, "cw_rope_append: type %u (f32, f16 or bf16)", p->type);
    CW_CHECK(p->layout <= CW_ROPE_INTERLEAVED, CW_ERR_INVALID_ARG, "cw_rope_append: layout %u",
             p->layout);
    CW_CHECK(p->n_tokens > 0 && p->n_tokens < (1u << 31) && p->n_heads <= 4096 &&
                 p->n_kv <= 4096 && p->n_heads + p->n_kv > 0 && p->head_dim > 0 &&
                 p->head_dim <= 1024,
             CW_ERR_INVALID_ARG, "cw_rope_append: bad shape");
    const size_t es = p->type == CW_GGUF_F32 ? 4 : 2, T = p->n_tokens, D = p->head_dim;
    const uint64_t big = 1ull << 40;  // keeps the byte counts below from overflowing
    CW_CHECK(p->q_off < big && p->k_off < big && p->v_off < big && p->q_stride < (1ull << 30) &&
                 p->k_stride < (1ull << 30) && p->v_stride < (1ull << 30),
             CW_ERR_INVALID_ARG, "cw_rope_append: bad offset or stride");
    BufEntry *plan, *pos, *q = nullptr, *qo = nullptr, *k = nullptr, *v = nullptr, *slots = nullptr,
                          *kc = nullptr, *vc = nullptr;
    CW_TRY(buf_get(ctx, p->plan, &plan, 0, "cw_rope_append(plan)"));
    CW_CHECK(plan->rope_dim, CW_ERR_INVALID_ARG, "cw_rope_append: not a plan of cw_rope_plan");
    CW_CHECK(plan->rope_dim <= D, CW_ERR_INVALID_ARG,
             "cw_rope_append: the plan rotates %u of %zu elements", plan->rope_dim, D);
    CW_TRY(buf_get(ctx, p->positions, &pos, T * 4, "cw_rope_append(positions)"));
    RopeArgs a{};
    if (p->n_heads) {
        const size_t w = p->n_heads * D;
        CW_CHECK(p->q_stride >= w || T == 1, CW_ERR_INVALID_ARG, "cw_rope_append: q_stride");
        CW_TRY(buf_get(ctx, p->q, &q, (p->q_off + (T - 1) * p->q_stride + w) * es,
                       "cw_rope_append(q)"));
        CW_TRY(buf_get(ctx, p->q_out, &qo, T * w * es, "cw_rope_append(q_out)"));
        CW_CHECK(q->ptr != qo->ptr || (p->q_off == 0 && (p->q_stride == w || T == 1)),
                 CW_ERR_INVALID_ARG, "cw_rope_append: q in place needs contiguous rows");
        a.q = (const char*)q->ptr + p->q_off * es;
        a.q_out = qo->ptr;
    }
    if (p->n_kv) {
        const size_t w = p->n_kv * D;
        CW_CHECK((p->k_stride >= w && p->v_stride >= w) || T == 1, CW_ERR_INVALID_ARG,
                 "cw_rope_append: k_stride, v_stride");
        CW_CHECK(p->page_size > 0 && p->page_size <= (1u << 20) && p->n_pages > 0 &&
                     (uint64_t)p->n_pages * p->page_size < (1ull << 31),
                 CW_ERR_INVALID_ARG, "cw_rope_append: bad cache shape");
        CW_TRY(buf_get(ctx, p->k, &k, (p->k_off + (T - 1) * p->k_stride + w) * es,
                       "cw_rope_append(k)"));
        CW_TRY(buf_get(ctx, p->v, &v, (p->v_off + (T - 1) * p->v_stride + w) * es,
                       "cw_rope_append(v)"));
        CW_TRY(buf_get(ctx, p->slots, &slots, T * 4, "cw_rope_append(slots)"));
        const size_t cache = (size_t)p->n_pages * p->page_size * w * es;
        CW_TRY(buf_get(ctx, p->k_cache, &kc, cache, "cw_rope_append(k_cache)"));
        CW_TRY(buf_get(ctx, p->v_cache, &vc, cache, "cw_rope_append(v_cache)"));
        a.k = (const char*)k->ptr + p->k_off * es;
        a.v = (const char*)v->ptr + p->v_off * es;
        a.slots = (const int*)slots->ptr;
        a.k_cache = kc->ptr;
        a.v_cache = vc->ptr;
        a.page = (int)p->page_size;
        a.n_slots = (long long)p->n_pages * p->page_size;
    }
    a.steps = (const unsigned long long*)plan->ptr;
    a.amp = plan->rope_amp;
    a.positions = (const int*)pos->ptr;
    a.q_stride = (long long)p->q_stride;
    a.k_stride = (long long)p->k_stride;
    a.v_stride = (long long)p->v_stride;
    a.rot = (int)plan->rope_dim;
    a.n_tokens = (int)T;
    a.H = (int)p->n_heads;
    a.K = (int)p->n_kv;
    a.D = (int)D;
    a.status = ctx->d_status;
    // the widest vector that divides the rotated halves, the rows and their places
    const uint64_t every = (uint64_t)(a.rot / 2) | D | (p->n_heads ? p->q_off | p->q_stride : 0) |
                           (p->n_kv ? p->k_off | p->k_stride | p->v_off | p->v_stride : 0);
    const uint64_t vec = std::min<uint64_t>(every & (~every + 1), 16 / es);
    cudaSetDevice(ctx->device);
    OpScope scope(ctx, "rope_append");
    const bool half = p->layout == CW_ROPE_HALF;
    auto go = [&](auto tag) -> int {
        typedef decltype(tag) T_;
        if constexpr (sizeof(T_) == 2)
            if (vec == 8) return rope_launch<T_, 8>(ctx, a, half);
        if (vec == 4) return rope_launch<T_, 4>(ctx, a, half);
        if (vec == 2) return rope_launch<T_, 2>(ctx, a, half);
        return rope_launch<T_, 1>(ctx, a, half);
    };
    if (p->type == CW_GGUF_F32) return go(float());
    if (p->type == CW_GGUF_F16) return go(__half());
    return go(__nv_bfloat16());
}

}  // extern "C"
