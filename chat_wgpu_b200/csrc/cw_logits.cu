// cw_logits.cu -- penalties for repeated tokens, biases and grammar masks on rows of
// logits, and the argmax of the result (cw_adjust_logits).
//
//   x -> x / rep or x rep (seen)  -> (x - freq n) - pres (n > 0)  -> + bias  -> -inf (masked)
//
// Memory bound: a row is read and written once.  A cluster of CTAs takes a row, each a
// slice of the vocabulary.  A CTA first goes through the row's whole history and counts
// the tokens of its own slice in shared memory (whole-number atomics, so their order does
// not matter; the history is short and comes from L2 after the first CTA), and notes the
// last bias entry of each.  Then it streams its slice.  The argmax is joined over the
// cluster through distributed shared memory: no word outside the row's own outputs is
// written, so calls and graph replays share nothing.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

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
    int slice;  // vocabulary entries of a CTA's slice, a multiple of 16
    int* status;
};

constexpr int LG_THREADS = 512;
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
__global__ void __launch_bounds__(LG_THREADS) k_adjust_logits(const __grid_constant__ LogitArgs a) {
    constexpr int VEC = WIDE ? 16 / sizeof(T) : 1;
    typedef typename VecOf<VEC * sizeof(T)>::type V;
    union Pack {
        V v;
        T e[VEC];
    };
    extern __shared__ __align__(16) uint32_t sm[];
    __shared__ unsigned long long s_key[LG_THREADS / 32], s_all[16];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (a.best) cluster.barrier_arrive();  // waited for before a CTA writes to another's memory
    const int tid = threadIdx.x, r = blockIdx.y, cta = blockIdx.x, ctas = gridDim.x;
    uint32_t* s_count = sm;            // [slice]
    uint32_t* s_bias = sm + a.slice;   // [slice] last entry of the token, counted from 1
    pdl_wait();
    const T* in = (const T*)a.logits + r * a.stride;
    T* out = (T*)a.out + (long long)r * a.vocab;
    const int shift = WIDE ? (int)(((uintptr_t)in & 15) / sizeof(T)) : 0;
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
    const uint32_t* mask = nullptr;
    if (a.masks) {
        const int m = a.mask_rows ? a.mask_rows[r] : r;
        if (m >= a.n_masks) {
            if (cta == 0 && tid == 0) lg_bad(a);
        } else if (m >= 0) {
            mask = a.masks + (size_t)m * a.words;
        }
    }
    const bool hist = h1 > h0, bias = b1 > b0;
    float top = -3.402823e38f;
    unsigned at = 0;
    for (long long base = (long long)cta * a.slice; base < (long long)a.vocab + shift;
         base += (long long)ctas * a.slice) {
        const int u0 = (int)base, u1 = (int)min(base + a.slice, (long long)a.vocab + shift);
        if (hist || bias) {
            __syncthreads();  // the slice before has been read
            for (int i = tid; i < a.slice / 4; i += LG_THREADS) {
                if (hist) ((uint4*)s_count)[i] = make_uint4(0, 0, 0, 0);
                if (bias) ((uint4*)s_bias)[i] = make_uint4(0, 0, 0, 0);
            }
            __syncthreads();
            for (int i = h0 + tid; i < h1; i += LG_THREADS) {
                const int t = a.tokens[i];
                if (t < 0 || t >= a.vocab) {
                    if (cta == 0) lg_bad(a);
                    continue;
                }
                const int u = t + shift;
                if (u < u0 || u >= u1) continue;
                if (i - h0 < lead) atomicOr(&s_count[u - u0], LG_LED);
                else atomicAdd(&s_count[u - u0], 1u);
            }
            for (int i = b0 + tid; i < b1; i += LG_THREADS) {
                const int t = a.bias_tokens[i];
                if (t < 0 || t >= a.vocab) {
                    if (cta == 0) lg_bad(a);
                    continue;
                }
                const int u = t + shift;
                if (u >= u0 && u < u1) atomicMax(&s_bias[u - u0], (unsigned)(i - b0) + 1u);
            }
            __syncthreads();
        }
        // one logit; each step is rounded by itself, as the definition says
        auto adjust = [&](T x, int u) {
            float y = rp_f32(x);
            if (hist) {
                const uint32_t c = s_count[u - u0];
                if (c) {
                    y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                    const uint32_t n = c & ~LG_LED;
                    if (n) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, (float)n)), pres);
                }
            }
            if (bias) {
                const uint32_t i = s_bias[u - u0];
                if (i) y = __fadd_rn(y, a.bias_values[b0 + (int)i - 1]);
            }
            if (mask) {
                const int v = u - shift;
                if (!(mask[v >> 5] >> (v & 31) & 1)) y = -INFINITY;
            }
            T z;
            rp_set(&z, y);
            y = rp_f32(z);
            if (y > top) {  // positions ascend in a thread: the lowest of equals stays
                top = y;
                at = (unsigned)(u - shift);
            }
            return z;
        };
        for (int u = u0 + tid * VEC; u < u1; u += LG_THREADS * VEC) {
            if (u >= shift && u + VEC <= a.vocab + shift) {
                Pack p;
                p.v = *(const V*)(in + (u - shift));
#pragma unroll
                for (int i = 0; i < VEC; i++) p.e[i] = adjust(p.e[i], u + i);
                *(V*)(out + (u - shift)) = p.v;
            } else {
                for (int i = 0; i < VEC; i++)
                    if (u + i >= shift && u + i < a.vocab + shift)
                        out[u + i - shift] = adjust(in[u + i - shift], u + i);
            }
        }
    }
    pdl_trigger();
    if (!a.best) return;
    unsigned long long key = argmax_key_init();
    if (top > -3.402823e38f) key = argmax_key(top, at);
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
    // up to 16 CTAs to a row (one cluster), no slice shorter than a pass of the threads
    const int span = a.vocab + 16, ctas = std::max(1, std::min(16, span / (LG_THREADS * 4)));
    const int most = a.bias_starts ? 24 * 1024 : 48 * 1024;  // 192 KB of shared memory
    a.slice = std::min(most, ((span + ctas - 1) / ctas + 15) / 16 * 16);
    const size_t smem = (size_t)a.slice * 4 * (a.bias_starts ? 2 : a.penalties ? 1 : 0);
    CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 192 * 1024));
    CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
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
