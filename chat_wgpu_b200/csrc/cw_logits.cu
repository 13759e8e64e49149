// cw_logits.cu -- penalties for repeated tokens, biases and grammar masks on rows of
// logits, and the argmax of the result (cw_adjust_logits).
//
//   x -> x / rep or x rep (seen)  -> (x - freq n) - pres (n > 0)  -> + bias  -> -inf (masked)
//
// Memory bound: a row is read and written once, but for logits in 16 bytes of which no
// token is allowed, which are not read.  A cluster of CTAs takes a row, each a slice of the
// vocabulary.  A CTA asks for its first logits, then goes through the row's whole lists and
// counts the tokens of its own slice in shared memory (whole-number atomics, so their order
// does not matter; the lists are short and come from L2 after the first CTA).  A bit for each
// listed token says where to look, and the number of bits before it where its count and its
// last bias entry are: memory goes by the lists' length, not by the vocabulary's.  Then it
// streams its slice, 8 or 4 logits to a look at the bits.  The argmax is joined over the cluster through distributed
// shared memory: no word outside the row's own outputs is written, so calls and graph
// replays share nothing.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <limits.h>

#include <algorithm>

#include "cw_common.h"
#include "cw_rotary.cuh"

namespace cw {

struct LogitArgs {
    const void* logits;
    void* out;
    const float* penalties;
    const int *tokens, *starts, *prompts, *bias_tokens, *bias_starts, *mask_rows;
    const float* bias_values;
    const uint32_t* masks;
    uint32_t* best;
    long long stride;
    int n_rows, vocab, n_tokens, n_bias, n_masks, words;
    int slice;  // vocabulary entries of a CTA's slice, a multiple of 32
    int* status;
};

constexpr int LG_THREADS = 512;
constexpr int LG_DEEP = 3;  // 16-byte vectors of a thread in flight
constexpr int LG_TOKENS = 4096;  // distinct tokens of a row's lists in a slice that there is room for
constexpr uint32_t LG_LED = 1u << 31;  // in the history's prompt part; the low bits count the rest

__device__ __forceinline__ void lg_bad(const LogitArgs& a) {
    atomicCAS(a.status, DEV_OK, DEV_BAD_INPUT);
}
// List r of ragged lists: [x, y) of n entries.
__device__ __forceinline__ void lg_list(const LogitArgs& a, const int* starts, int r, int n, int& x,
                                        int& y, bool report) {
    const int s0 = starts[r], s1 = starts[r + 1];
    x = min(max(s0, 0), n);
    y = min(max(s1, x), n);
    if (report && (x != s0 || y != s1)) lg_bad(a);
}

// VEC elements of 16 bytes where in and out rows have the same alignment, else one by one.
// Positions u count from the 16-byte boundary at or before the row's first logit: logit
// v is at u = v + shift, and slices and vectors start at multiples of VEC.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(LG_THREADS, 2) k_adjust_logits(const __grid_constant__ LogitArgs a) {
    constexpr int VEC = WIDE ? 16 / sizeof(T) : 1;
    constexpr uint32_t EVERY = (1u << VEC) - 1;
    typedef typename VecOf<VEC * sizeof(T)>::type V;
    union Pack {
        V v;
        T e[VEC];
    };
    extern __shared__ __align__(16) uint32_t sm[];
    __shared__ unsigned long long s_key[LG_THREADS / 32], s_all[16];
    __shared__ int s_sum[LG_THREADS / 32], s_n;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (a.best) cluster.barrier_arrive();  // waited for before a CTA writes to another's memory
    const int tid = threadIdx.x, r = blockIdx.y, cta = blockIdx.x, ctas = gridDim.x;
    const int words = a.slice / 32;
    uint32_t* s_bits = sm;                // [words] the token is in one of the lists
    uint32_t* s_rank = s_bits + words;    // [words] bits set before the word
    uint32_t* s_count = s_rank + words;   // [LG_TOKENS] of the listed tokens, in order
    int* s_place = (int*)s_count + LG_TOKENS;  // where they are in the slice
    uint32_t* s_mine = s_count + 2 * LG_TOKENS;  // the history's tokens that lie here, if few
    uint32_t* s_last = s_count + 3 * LG_TOKENS;  // and their last bias entry, counted from 1
    pdl_wait();
    pdl_trigger();
    const T* in = (const T*)a.logits + r * a.stride;
    T* out = (T*)a.out + (long long)r * a.vocab;
    const int shift = WIDE ? (int)(((uintptr_t)in & 15) / sizeof(T)) : 0;
    const int end = a.vocab + shift;
    const uint32_t* mask = nullptr;
    if (a.masks) {
        const int m = a.mask_rows ? a.mask_rows[r] : r;
        if (m >= a.n_masks) {
            if (cta == 0 && tid == 0) lg_bad(a);
        } else if (m >= 0) {
            mask = a.masks + (size_t)m * a.words;
        }
    }
    // which of the VEC tokens from position u (all in the vocabulary) are allowed
    auto allowed = [&](int u) -> uint32_t {
        if (!mask) return EVERY;
        const int v = u - shift, w = v >> 5, x = v & 31;
        uint32_t bits = mask[w] >> x;
        if (x + VEC > 32) bits |= mask[w + 1] << (32 - x);
        return bits & EVERY;
    };
    auto whole = [&](int u) { return u >= shift && u + VEC <= end; };
    // a thread's next LG_DEEP vectors; one without an allowed token is not read
    Pack p[LG_DEEP];
    uint32_t on[LG_DEEP];
    auto load = [&](int u, int u1) {
#pragma unroll
        for (int i = 0; i < LG_DEEP; i++) {
            const int x = u + i * LG_THREADS * VEC;
            on[i] = x < u1 && whole(x) ? allowed(x) : 0;
        }
#pragma unroll
        for (int i = 0; i < LG_DEEP; i++)
            if (on[i]) p[i].v = *(const V*)(in + (u + i * LG_THREADS * VEC - shift));
    };
    const int first = cta * a.slice;
    load(first + tid * VEC, min(first + a.slice, end));  // in flight while the lists are read
    float rep = 1.f, freq = 0.f, pres = 0.f;
    int h0 = 0, h1 = 0, lead = 0, b0 = 0, b1 = 0;
    if (a.penalties) {
        rep = a.penalties[3 * r];
        freq = a.penalties[3 * r + 1];
        pres = a.penalties[3 * r + 2];
        lg_list(a, a.starts, r, a.n_tokens, h0, h1, cta == 0 && tid == 0);
        lead = a.prompts ? min(max(a.prompts[r], 0), h1 - h0) : 0;
        if (rep == 1.f && freq == 0.f && pres == 0.f) h1 = h0;
    }
    if (a.bias_starts) lg_list(a, a.bias_starts, r, a.n_bias, b0, b1, cta == 0 && tid == 0);
    const bool hist = h1 > h0, bias = b1 > b0;
    float top = -3.402823e38f;
    unsigned at = 0;
    // f(place in [u0, u1), entry) for the tokens [x, y) of a list that lie there
    int u0 = 0, u1 = 0;
    auto each = [&](const int* tokens, int x, int y, auto f) {
        for (int i = x + tid; i < y; i += 8 * LG_THREADS) {
            int t[8];
#pragma unroll
            for (int k = 0; k < 8; k++)
                t[k] = i + k * LG_THREADS < y ? tokens[i + k * LG_THREADS] : INT_MAX;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if (i + k * LG_THREADS >= y) break;
                const unsigned j = (unsigned)t[k] + (unsigned)shift - (unsigned)u0;
                if (j < (unsigned)(u1 - u0) && t[k] >= 0) f((int)j, i + k * LG_THREADS);
                else if (cta == 0 && (unsigned)t[k] >= (unsigned)a.vocab) lg_bad(a);
            }
        }
    };
    auto rank = [&](int j) {  // which of the listed tokens the one at place j is
        return s_rank[j >> 5] + __popc(s_bits[j >> 5] & ((1u << (j & 31)) - 1));
    };
    int step = a.slice;  // entries at a time
    bool loaded = true;  // the first vectors are there
    // pieces of the CTA's slices (positions stay below 2^30 + 16, sums of two below 2^31)
    for (int slice0 = first, base = first; base < end;) {
        u0 = base;
        u1 = min(min(slice0 + a.slice, end), u0 + step);
        int n_listed = 0;
        if (hist || bias) {
            __syncthreads();  // what went before has been read
            for (int i = tid; i < words; i += LG_THREADS) s_bits[i] = 0;
            if (tid == 0) s_n = 0;
            __syncthreads();
            auto mark = [&](int j, int) {
                const uint32_t bit = 1u << (j & 31);
                if (!(*(volatile uint32_t*)&s_bits[j >> 5] & bit)) atomicOr(&s_bits[j >> 5], bit);
            };
            each(a.tokens, h0, h1, [&](int j, int i) {
                mark(j, i);
                // kept for the count, so that it need not go through the history again
                const unsigned among = __activemask();
                const int first = __ffs(among) - 1, mine = __popc(among & ((1u << (tid & 31)) - 1));
                int k = 0;
                if ((tid & 31) == first) k = atomicAdd(&s_n, __popc(among));
                k = __shfl_sync(among, k, first) + mine;
                if (k < LG_TOKENS) s_mine[k] = (uint32_t)j | (i - h0 < lead ? LG_LED : 0u);
            });
            each(a.bias_tokens, b0, b1, mark);
            __syncthreads();
            // ranks: a thread's words, then its place among the threads
            const int per = (words + LG_THREADS - 1) / LG_THREADS;
            int mine = 0;
            for (int i = tid * per; i < min(words, tid * per + per); i++) mine += __popc(s_bits[i]);
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(FULL, incl, o);
                if ((tid & 31) >= o) incl += x;
            }
            if ((tid & 31) == 31) s_sum[tid >> 5] = incl;
            __syncthreads();
            int before = 0, total = 0;
            for (int w = 0; w < LG_THREADS / 32; w++) {
                if (w == tid >> 5) before = total;
                total += s_sum[w];
            }
            if (total > LG_TOKENS) {  // more listed tokens than there is room for: in pieces
                step = LG_TOKENS;
                loaded = false;
                continue;
            }
            before += incl - mine;
            for (int i = tid * per; i < min(words, tid * per + per); i++) {
                s_rank[i] = before;
                before += __popc(s_bits[i]);
            }
            for (int i = tid; i < total; i += LG_THREADS) {
                s_count[i] = 0;
                if (a.bias_starts) s_last[i] = 0;
            }
            __syncthreads();
            auto count = [&](int j, bool led) {
                const int k = rank(j);
                s_place[k] = j;
                if (led) atomicOr(&s_count[k], LG_LED);
                else atomicAdd(&s_count[k], 1u);
            };
            if (s_n <= LG_TOKENS) {
                for (int i = tid; i < s_n; i += LG_THREADS)
                    count((int)(s_mine[i] & ~LG_LED), (s_mine[i] & LG_LED) != 0);
            } else {
                each(a.tokens, h0, h1, [&](int j, int i) { count(j, i - h0 < lead); });
            }
            each(a.bias_tokens, b0, b1, [&](int j, int i) {
                const int k = rank(j);
                s_place[k] = j;
                atomicMax(&s_last[k], (unsigned)(i - b0) + 1u);
            });
            n_listed = total;
            __syncthreads();
        }
        auto listed = [&](int u) -> uint32_t {  // of the VEC tokens from position u
            if (!hist && !bias) return 0;
            return s_bits[(u - u0) >> 5] >> ((u - u0) & 31) & EVERY;
        };
        auto is_on = [&](int v) { return !mask || (mask[v >> 5] >> (v & 31) & 1); };
        auto better = [&](float y, int v) {  // the lowest index of equals
            if (y > top || (y == top && (unsigned)v < at)) {
                top = y;
                at = (unsigned)v;
            }
        };
        // ---- all tokens as if none was listed; the listed ones are left out of the argmax
        float most = -INFINITY;  // of the thread's vectors
        int where = -1;
        for (int u = u0 + tid * VEC; u < u1; u += LG_DEEP * LG_THREADS * VEC) {
            if (!loaded) load(u, u1);
            loaded = false;
#pragma unroll
            for (int i = 0; i < LG_DEEP; i++) {
                const int x = u + i * LG_THREADS * VEC;
                if (x >= u1) break;
                if (!whole(x)) {  // the row's ends
                    for (int j = max(x, shift); j < min(x + VEC, end); j++) {
                        const int v = j - shift;
                        T z = in[v];
                        if (!is_on(v)) rp_set(&z, -INFINITY);
                        else if (!((hist || bias) && (s_bits[(j - u0) >> 5] >> ((j - u0) & 31) & 1)))
                            better(rp_f32(z), v);
                        out[v] = z;
                    }
                    continue;
                }
                if (on[i] != EVERY) {
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                        if (!(on[i] >> j & 1)) rp_set(&p[i].e[j], -INFINITY);
                }
                if (on[i] != EVERY || a.out != a.logits) *(V*)(out + (x - shift)) = p[i].v;
                if (!a.best) continue;
                const uint32_t list = listed(x);
                if (list) {
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                        if (list >> j & 1) rp_set(&p[i].e[j], -INFINITY);
                }
                float m = rp_f32(p[i].e[0]);
#pragma unroll
                for (int j = 1; j < VEC; j++) m = fmaxf(m, rp_f32(p[i].e[j]));
                if (m > most) {  // positions ascend: the first of equal vectors
                    most = m;
                    where = x;
                }
            }
        }
        if (where >= 0) {  // which of its tokens it was
            Pack q;
            q.v = *(const V*)(out + (where - shift));
            const uint32_t list = listed(where);
#pragma unroll
            for (int j = VEC - 1; j >= 0; j--)
                if (!(list >> j & 1) && rp_f32(q.e[j]) == most) better(most, where + j - shift);
        }
        // ---- the listed ones; each step is rounded by itself, as the definition says
        if (n_listed) __syncthreads();
        for (int k = tid; k < n_listed; k += LG_THREADS) {
            const int v = s_place[k] + u0 - shift;
            if (!is_on(v)) continue;
            float y = rp_f32(in[v]);
            const uint32_t c = hist ? s_count[k] : 0, e = bias ? s_last[k] : 0;
            if (c) {
                y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                const uint32_t n = c & ~LG_LED;
                if (n) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, (float)n)), pres);
            }
            if (e) y = __fadd_rn(y, a.bias_values[b0 + (int)e - 1]);
            T z;
            rp_set(&z, y);
            better(rp_f32(z), v);
            out[v] = z;
        }
        loaded = false;
        base = u1;
        if (u1 == slice0 + a.slice) base = slice0 += ctas * a.slice;
    }
    if (!a.best) return;
    unsigned long long key = argmax_key_init();
    if (top > -3.402823e38f) key = argmax_key(top, at);  // else index 0
    for (int o = 16; o; o >>= 1) {
        const unsigned long long x = __shfl_xor_sync(FULL, key, o);
        key = x > key ? x : key;
    }
    if ((tid & 31) == 0) s_key[tid >> 5] = key;
    __syncthreads();
    if (tid == 0) {
        for (int i = 0; i < LG_THREADS / 32; i++) key = s_key[i] > key ? s_key[i] : key;
    }
    cluster.barrier_wait();
    if (tid == 0) *cluster.map_shared_rank(&s_all[cta], 0) = key;
    cluster.sync();
    if (cta == 0 && tid == 0) {
        for (int i = 0; i < ctas; i++) key = s_all[i] > key ? s_all[i] : key;
        a.best[r] = argmax_key_index(key);
    }
}

template <typename T> static int adjust_launch(cw_ctx* ctx, LogitArgs& a, bool wide) {
    auto kern = wide ? k_adjust_logits<T, true> : k_adjust_logits<T, false>;
    // up to 16 CTAs to a row (one cluster), no slice shorter than a pass of the threads; with
    // many rows fewer, so that a row's lists are gone through less often (256 rows of 151936: 61
    // us with two CTAs to a row, 74 with four, 65 with one)
    const int span = a.vocab + 16, many = std::max(1, 4 * ctx->sm_count / a.n_rows);
    const int ctas = std::max(1, std::min({16, many, span / (LG_THREADS * 4)}));
    a.slice = std::min(128 * 1024, ((span + ctas - 1) / ctas + 31) / 32 * 32);
    const bool lists = a.penalties || a.bias_starts;
    const size_t smem = lists ? a.slice / 4 + (size_t)LG_TOKENS * 4 * (a.bias_starts ? 4 : 3) : 0;
    static bool set[2][64] = {};
    if (!set[wide][ctx->device & 63]) {
        CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024));
        CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        set[wide][ctx->device & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, a.n_rows);
    cfg.blockDim = dim3(LG_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CW_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
    return check_launch("adjust_logits");
}

}  // namespace cw

using namespace cw;

extern "C" int cw_adjust_logits(cw_ctx* ctx, const cw_adjust_logits_args* p) {
    clear_error();
    CW_CHECK(ctx && p, CW_ERR_INVALID_ARG, "cw_adjust_logits: bad arguments");
    CW_CHECK(p->type == CW_GGUF_F32 || p->type == CW_GGUF_F16 || p->type == CW_GGUF_BF16,
             CW_ERR_UNSUPPORTED, "cw_adjust_logits: type %u (f32, f16 or bf16)", p->type);
    CW_CHECK(p->n_rows > 0 && p->n_rows <= 65535 && p->vocab > 0 && p->vocab < (1u << 30) &&
                 p->n_tokens < (1u << 30) && p->n_bias < (1u << 30) && p->n_masks < (1u << 30),
             CW_ERR_INVALID_ARG, "cw_adjust_logits: bad shape");
    CW_CHECK((p->stride >= p->vocab || p->n_rows == 1) && p->stride < (1ull << 32) &&
                 p->off < (1ull << 40),
             CW_ERR_INVALID_ARG, "cw_adjust_logits: bad offset or stride");
    const size_t es = p->type == CW_GGUF_F32 ? 4 : 2, R = p->n_rows, V = p->vocab;
    LogitArgs a{};
    BufEntry* e;
    struct Span {
        const char* at;
        size_t n;
        const char* what;
    } in[12];
    int ins = 0;
    auto get = [&](cw_buf b, size_t n, auto** to, const char* what) -> int {
        CW_TRY(buf_get(ctx, b, &e, n, what));
        *to = (std::remove_reference_t<decltype(*to)>)e->ptr;
        in[ins++] = {(const char*)e->ptr, n, what};
        return CW_OK;
    };
    CW_TRY(buf_get(ctx, p->logits, &e, (p->off + (R - 1) * p->stride + V) * es,
                   "cw_adjust_logits(logits)"));
    a.logits = (const char*)e->ptr + p->off * es;
    const size_t n_in = ((R - 1) * p->stride + V) * es;
    if (p->penalties) {
        CW_TRY(get(p->penalties, R * 12, &a.penalties, "cw_adjust_logits(penalties)"));
        CW_TRY(get(p->starts, (R + 1) * 4, &a.starts, "cw_adjust_logits(starts)"));
        if (p->n_tokens)
            CW_TRY(get(p->tokens, (size_t)p->n_tokens * 4, &a.tokens, "cw_adjust_logits(tokens)"));
        if (p->prompts) CW_TRY(get(p->prompts, R * 4, &a.prompts, "cw_adjust_logits(prompts)"));
    }
    if (p->bias_starts) {
        CW_TRY(get(p->bias_starts, (R + 1) * 4, &a.bias_starts, "cw_adjust_logits(bias_starts)"));
        if (p->n_bias) {
            CW_TRY(get(p->bias_tokens, (size_t)p->n_bias * 4, &a.bias_tokens,
                       "cw_adjust_logits(bias_tokens)"));
            CW_TRY(get(p->bias_values, (size_t)p->n_bias * 4, &a.bias_values,
                       "cw_adjust_logits(bias_values)"));
        }
    }
    a.words = (int)((V + 31) / 32);
    if (p->masks) {
        CW_CHECK(p->n_masks > 0 && (p->mask_rows || p->n_masks >= R), CW_ERR_INVALID_ARG,
                 "cw_adjust_logits: %u masks for %zu rows", p->n_masks, R);
        CW_TRY(get(p->masks, (size_t)p->n_masks * a.words * 4, &a.masks,
                   "cw_adjust_logits(masks)"));
        if (p->mask_rows)
            CW_TRY(get(p->mask_rows, R * 4, &a.mask_rows, "cw_adjust_logits(mask_rows)"));
    }
    const int reads = ins;
    CW_TRY(buf_get(ctx, p->out, &e, R * V * es, "cw_adjust_logits(out)"));
    a.out = e->ptr;
    for (int i = 0; i < reads; i++)
        CW_CHECK(!spans_meet(a.out, R * V * es, in[i].at, in[i].n), CW_ERR_INVALID_ARG,
                 "cw_adjust_logits(out) lies on %s", in[i].what);
    CW_CHECK((a.out == a.logits && (p->stride == V || R == 1)) ||
                 !spans_meet(a.out, R * V * es, a.logits, n_in),
             CW_ERR_INVALID_ARG, "cw_adjust_logits(out) lies on the logits");
    if (p->best) {
        CW_TRY(buf_get(ctx, p->best, &e, R * 4, "cw_adjust_logits(best)"));
        a.best = (uint32_t*)e->ptr;
        for (int i = 0; i < reads; i++)
            CW_CHECK(!spans_meet(a.best, R * 4, in[i].at, in[i].n), CW_ERR_INVALID_ARG,
                     "cw_adjust_logits(best) lies on %s", in[i].what);
        CW_CHECK(!spans_meet(a.best, R * 4, a.logits, n_in) &&
                     !spans_meet(a.best, R * 4, a.out, R * V * es),
                 CW_ERR_INVALID_ARG, "cw_adjust_logits(best) lies on the logits or out");
    }
    a.stride = (long long)p->stride;
    a.n_rows = (int)R;
    a.vocab = (int)V;
    a.n_tokens = (int)p->n_tokens;
    a.n_bias = (int)p->n_bias;
    a.n_masks = (int)p->n_masks;
    a.status = ctx->d_status;
    // vectors where every row lies the same way in both buffers
    const bool wide = (((uintptr_t)a.logits ^ (uintptr_t)a.out) & 15) == 0 &&
                      (R == 1 || (p->stride - V) * es % 16 == 0);
    cudaSetDevice(ctx->device);
    OpScope scope(ctx, "adjust_logits");
    if (p->type == CW_GGUF_F32) return adjust_launch<float>(ctx, a, wide);
    if (p->type == CW_GGUF_F16) return adjust_launch<__half>(ctx, a, wide);
    return adjust_launch<__nv_bfloat16>(ctx, a, wide);
}
