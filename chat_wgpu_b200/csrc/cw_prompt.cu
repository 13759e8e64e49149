// cw_prompt.cu -- causal attention of packed prompts (cw_prompt_attention): the entry
// point, and the kernel for every type, alignment and head size in f32 products.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,   w_ij = exp(cap(scale q_i . k_j) - m_i)
//
// Keys come in tiles; a row keeps its running maximum m_i, sum and weighted values, and
// scales the latter two when the maximum grows.  256 threads hold 64 x 64 scores as 4 x 4
// blocks and 64 x D sums as 4 rows by D / 16 columns.  It takes what the tensor cores do not:
// short f32 prompts (17 tokens of 16/8 heads in 9.5 us, of which its launch is 3), few f32
// rows over many keys (eight after 500 in 27 us), f32 past 128 dims (4000 tokens of 8/4 heads
// of 256 in 2.15 ms: 31 TFLOP/s, bound by the latency of its reads, two warps to a scheduler),
// 16-bit rows at odd places, and requests whose f32 values do not fit pairs.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "cw_prompt.cuh"

namespace cw {

constexpr int PF_ROWS = 64, PF_KEYS = PF_ROWS, PF_THREADS = 256;

// Fills [64][DP + 4] from row(m), zeros where it is null and past D: eight reads in flight (a
// row of 4000 keys one read at a time took 980 us), each of four elements where rows allow
// it (`wide`: D, strides and addresses are multiples).  Whether what this thread read is finite.
template <typename T, int DP, int N, typename F>
__device__ __forceinline__ bool pf_fill_by(float* to, int D, F row) {
    struct alignas(N * sizeof(T)) Vec {
        T e[N];
    };
    constexpr int PER = DP / N, ALL = PF_ROWS * PER, DEEP = ALL / PF_THREADS < 8 ? ALL / PF_THREADS : 8;
    bool odd = false;
    for (int i0 = threadIdx.x; i0 < ALL; i0 += DEEP * PF_THREADS) {
        Vec x[DEEP];
        bool on[DEEP];
#pragma unroll
        for (int e = 0; e < DEEP; e++) {
            const int i = i0 + e * PF_THREADS, d = i % PER * N;
            const T* from = row(i / PER);
            on[e] = from && d < D;
            if (on[e]) x[e] = *(const Vec*)(from + d);
        }
#pragma unroll
        for (int e = 0; e < DEEP; e++) {
            const int i = i0 + e * PF_THREADS, d = i % PER * N;
            alignas(16) float y[N];
#pragma unroll
            for (int n = 0; n < N; n++) {
                y[n] = on[e] ? pr_f32(x[e].e[n]) : 0.f;
                odd |= !isfinite(y[n]);
            }
            float* at = to + i / PER * (DP + 4) + d;
            if constexpr (N == 4) *(float4*)at = *(const float4*)y;
            else *at = y[0];
        }
    }
    return odd;
}
template <typename T, int DP, typename F>
__device__ __forceinline__ bool pf_fill(float* to, int D, bool wide, F row) {
    return wide ? pf_fill_by<T, DP, 4>(to, D, row) : pf_fill_by<T, DP, 1>(to, D, row);
}
// DP: head_dim rounded up to 64, 128 or 256.
template <typename T, int DP>
__global__ void __launch_bounds__(PF_THREADS) k_prompt(const __grid_constant__ PromptArgs a) {
    constexpr int LD = DP + 4, CN = DP / 16;
    extern __shared__ __align__(16) float sm[];
    float* sq = sm;                   // [PF_ROWS][LD]
    float* skv = sq + PF_ROWS * LD;   // [PF_KEYS][LD]
    float* sp = skv + PF_KEYS * LD;   // [PF_ROWS][PF_KEYS + 4]
    constexpr int LP = PF_KEYS + 4;
    const float log2e = 1.44269504088896341f;  // scores are in powers of two
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int warp_row = (tid >> 5) * 8;  // the warp's first row
    auto col = [&](int c) { return tx * 4 + c / 4 * 64 + c % 4; };  // the thread's dims
    const int head = blockIdx.x % a.K, block = blockIdx.x / a.K;
    pdl_wait();
    if (blockIdx.x == 0 && blockIdx.y == 0) prompt_check(a, tid, PF_THREADS);
    // the last blocks of a request have the most keys: they start first
    const PromptItem it = prompt_item(a, a.slots - 1 - block / ((a.bt * a.G + PF_ROWS - 1) / PF_ROWS));
    const int m0 = block % ((a.bt * a.G + PF_ROWS - 1) / PF_ROWS) * PF_ROWS;
    const int rows = min(PF_ROWS, it.rows * a.G - m0);
    if (rows <= 0 || (a.amax && !pr_odd(a, it.req, head))) return;
    const T* qb = (const T*)a.q + (long long)head * a.G * a.D;
    const T* kb = (const T*)a.k + (long long)it.key0 * a.k_stride + (long long)head * a.D;
    const T* vb = (const T*)a.v + (long long)it.key0 * a.v_stride + (long long)head * a.D;
    const bool wide = (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v) & (4 * sizeof(T) - 1)) == 0 &&
                      ((a.q_stride | a.k_stride | a.v_stride | a.D) & 3) == 0;
    (void)pf_fill<T, DP>(sq, a.D, wide, [&](int m) -> const T* {
        const int t = (m0 + m) / a.G, g = (m0 + m) - t * a.G;
        return m < rows ? qb + (long long)(it.row0 + t) * a.q_stride + g * a.D : nullptr;
    });
    float o[4][CN], top[4], sum[4];
    int lim[4], low[4];  // the row sees keys [low, lim]
#pragma unroll
    for (int i = 0; i < 4; i++) {
        top[i] = -INFINITY;
        sum[i] = 0.f;
#pragma unroll
        for (int c = 0; c < CN; c++) o[i][c] = 0.f;
        const int m = m0 + ty * 4 + i, t = m / a.G;
        lim[i] = ty * 4 + i < rows ? min(it.past + t, it.keys - 1) : -1;
        low[i] = a.window > 0 ? max(it.past + t - a.window + 1, 0) : 0;
    }
    int last = min(it.past + (m0 + rows - 1) / a.G, it.keys - 1);
    int first = it.first / PF_KEYS * PF_KEYS;
    if (gridDim.y > 1) {  // this block's share of the tiles
        const int tiles = last >= first ? (last - first) / PF_KEYS + 1 : 0;
        const int per = (tiles + gridDim.y - 1) / gridDim.y * PF_KEYS;
        first += blockIdx.y * per;
        last = min(last, first + per - 1);
    }
    // keys that every row of the block sees
    const int all1 = min(it.past + m0 / a.G, it.keys - 1);
    const int all0 = a.window > 0 ? it.past + (m0 + rows - 1) / a.G - a.window + 1 : 0;
    for (int kt = first; kt <= last; kt += PF_KEYS) {
        const bool mixed = kt < all0 || kt + PF_KEYS - 1 > all1;
        __syncthreads();
        (void)pf_fill<T, DP>(skv, a.D, wide, [&](int j) -> const T* {
            return kt + j <= last ? kb + (long long)(kt + j) * a.k_stride : nullptr;
        });
        __syncthreads();
        // of the tile only the keys there are, 16 to a column block, and only warps with rows
        // (asked inside the loop, it made a row block of 256 dims 14 % slower)
        const int keys = min(PF_KEYS, last - kt + 1);
        float s[4][4] = {};
        auto scores = [&](auto n) {
            for (int d = 0; d < a.D; d += 4) {
                float4 x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = *(const float4*)&sq[(ty * 4 + i) * LD + d];
#pragma unroll
                for (int j = 0; j < decltype(n)::value; j++) {
                    const float4 y = *(const float4*)&skv[(tx + 16 * j) * LD + d];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        s[i][j] = fmaf(x[i].x, y.x, s[i][j]);
                        s[i][j] = fmaf(x[i].y, y.y, s[i][j]);
                        s[i][j] = fmaf(x[i].z, y.z, s[i][j]);
                        s[i][j] = fmaf(x[i].w, y.w, s[i][j]);
                    }
                }
            }
        };
        if (warp_row >= rows) {
        } else if (keys > 32) {
            scores(std::integral_constant<int, 4>());
        } else {
            scores(std::integral_constant<int, 2>());
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float t = top[i];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float x = s[i][j] * (a.softcap > 0.f ? a.scale / a.softcap : a.scale * log2e);
                if (a.softcap > 0.f) x = a.softcap * tanhf(x) * log2e;  // (softcap * log2e may pass f32)
                const int key = kt + tx + 16 * j;
                if (key < low[i] || key > lim[i]) x = -INFINITY;
                s[i][j] = x;
                t = fmaxf(t, x);
            }
#pragma unroll
            for (int w = 8; w; w >>= 1) t = fmaxf(t, __shfl_xor_sync(FULL, t, w));
            // scores of -inf weigh nothing, whatever the maximum
            const float from = t == -INFINITY ? 0.f : t;
            const float fix = top[i] == -INFINITY ? 0.f : exp2f(top[i] - from);
            top[i] = t;
            float l = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float p = exp2f(s[i][j] - from);
                l += p;
                sp[(ty * 4 + i) * LP + tx + 16 * j] = p;
            }
#pragma unroll
            for (int w = 8; w; w >>= 1) l += __shfl_xor_sync(FULL, l, w);
            sum[i] = sum[i] * fix + l;
#pragma unroll
            for (int c = 0; c < CN; c++) o[i][c] *= fix;
        }
        __syncthreads();
        const bool odd = pf_fill<T, DP>(skv, a.D, wide, [&](int j) -> const T* {
            return kt + j <= last ? vb + (long long)(kt + j) * a.v_stride : nullptr;
        });
        // a value that is not finite counts only where it is seen
        const bool careful = __syncthreads_or(mixed && odd);
        // four keys at a time: past the last one weights and values are 0
        auto values = [&](auto strict) {
            for (int j0 = 0; j0 < keys; j0 += 4) {
                alignas(16) float p[4][4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *(float4*)p[i] = *(const float4*)&sp[(ty * 4 + i) * LP + j0];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    alignas(16) float y[CN];
#pragma unroll
                    for (int c = 0; c < CN; c += 4)
                        *(float4*)&y[c] = *(const float4*)&skv[(j0 + j) * LD + col(c)];
                    const int key = kt + j0 + j;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (decltype(strict)::value && (key < low[i] || key > lim[i])) continue;
#pragma unroll
                        for (int c = 0; c < CN; c++) o[i][c] = fmaf(p[i][j], y[c], o[i][c]);
                    }
                }
            }
        };
        if (warp_row >= rows) {
        } else if (careful) {
            values(std::true_type());
        } else {
            values(std::false_type());
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int m = ty * 4 + i;
        if (m >= rows) continue;
        if (gridDim.y > 1) {
            const size_t at = ((size_t)blockIdx.x * gridDim.y + blockIdx.y) * PF_ROWS + m;
            if (tx == 0) a.ml[at] = make_float2(top[i], last < first ? -1.f : sum[i]);
#pragma unroll
            for (int c = 0; c < CN; c++)
                if (col(c) < a.dp) a.part[at * a.dp + col(c)] = o[i][c];
            continue;
        }
        const int t = (m0 + m) / a.G, g = (m0 + m) - t * a.G;
        const float inv = sum[i] > 0.f || sum[i] != sum[i] ? 1.f / sum[i] : 0.f;
        T* out = (T*)a.out + ((long long)(it.row0 + t) * a.H + head * a.G + g) * a.D;
#pragma unroll
        for (int c = 0; c < CN; c++) {
            const int d = col(c);
            if (d < a.D) out[d] = pr_to<T>(inv == 0.f ? 0.f : o[i][c] * inv);
        }
    }
}

// Joins the shares of each block's rows, a warp per row.
template <typename T>
__global__ void __launch_bounds__(PF_THREADS)
    k_prompt_split_join(const __grid_constant__ PromptArgs a, int splits) {
    const int m = blockIdx.y * (PF_THREADS / 32) + (threadIdx.x >> 5);
    const int per = (a.bt * a.G + PF_ROWS - 1) / PF_ROWS;
    const int head = blockIdx.x % a.K, block = blockIdx.x / a.K;
    pdl_trigger();
    pdl_wait();
    const PromptItem it = prompt_item(a, a.slots - 1 - block / per);
    const int row = block % per * PF_ROWS + m;
    if (row >= it.rows * a.G) return;
    const int t = row / a.G, g = row - t * a.G;
    prompt_join_row(a, splits, (T*)a.out + ((long long)(it.row0 + t) * a.H + head * a.G + g) * a.D,
                    [&](int i) { return ((size_t)blockIdx.x * splits + i) * PF_ROWS + m; });
}

template <typename T, int DP> static int prompt_go(cw_ctx* ctx, PromptArgs& a) {
    auto kern = k_prompt<T, DP>;
    const size_t smem = ((size_t)(PF_ROWS + PF_KEYS) * (DP + 4) + PF_ROWS * (PF_KEYS + 4)) * 4;
    static bool set[64] = {};
    if (!set[ctx->device & 63]) {
        CW_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        set[ctx->device & 63] = true;
    }
    a.bt = std::max(1, PF_ROWS / a.G);
    a.slots = a.n_rows / a.bt + a.n_req;
    const long long grid = (long long)a.slots * ((a.bt * a.G + PF_ROWS - 1) / PF_ROWS) * a.K;
    CW_CHECK(grid < (1ll << 31), CW_ERR_UNSUPPORTED, "cw_prompt_attention: too many rows");
    // few blocks over many keys share them out, four tiles each at least (what is left of a
    // call on the tensor cores is rare, and whole)
    int splits = 1;
    if (!a.amax && grid < ctx->sm_count) {
        splits = (int)std::min<long long>({2ll * ctx->sm_count / grid, a.n_keys / (4 * PF_KEYS), 64});
        splits = std::max(splits, 1);
    }
    if (splits > 1) {
        a.dp = (a.D + 7) / 8 * 8;
        const size_t rows = (size_t)grid * splits * PF_ROWS;
        CW_TRY(stream_scratch(ctx, &ctx->prompt_scratch, &ctx->prompt_scratch_bytes,
                              rows * a.dp * 4 + rows * 8, "cw_prompt_attention"));
        a.part = (float*)ctx->prompt_scratch;
        a.ml = (float2*)(a.part + rows * a.dp);
    }
    CW_TRY(launch_pdl(ctx, true, kern, dim3((unsigned)grid, splits), dim3(PF_THREADS), smem, a));
    if (splits > 1)
        CW_TRY(launch_pdl(ctx, true, k_prompt_split_join<T>, dim3((unsigned)grid, PF_ROWS / (PF_THREADS / 32)),
                          dim3(PF_THREADS), 0, a, splits));
    return check_launch("prompt_attention");
}
template <typename T> static int prompt_dims(cw_ctx* ctx, PromptArgs& a) {
    if (a.D <= 64) return prompt_go<T, 64>(ctx, a);
    if (a.D <= 128) return prompt_go<T, 128>(ctx, a);
    return prompt_go<T, 256>(ctx, a);
}

}  // namespace cw

using namespace cw;

extern "C" int cw_prompt_attention(cw_ctx* ctx, const cw_prompt_attn_args* p) {
    clear_error();
    CW_CHECK(ctx && p, CW_ERR_INVALID_ARG, "cw_prompt_attention: bad arguments");
    CW_CHECK(p->type == CW_GGUF_F32 || p->type == CW_GGUF_F16 || p->type == CW_GGUF_BF16,
             CW_ERR_UNSUPPORTED, "cw_prompt_attention: type %u (f32, f16 or bf16)", p->type);
    CW_CHECK(p->n_req > 0 && p->n_req <= (1u << 20) && p->n_rows > 0 && p->n_rows <= (1u << 28) &&
                 p->n_keys > 0 && p->n_keys <= (1u << 28) && p->n_kv > 0 && p->n_heads <= 4096 &&
                 p->n_heads >= p->n_kv && p->n_heads % p->n_kv == 0 && p->head_dim > 0 &&
                 p->head_dim <= 256 && p->window < (1u << 31),
             CW_ERR_INVALID_ARG, "cw_prompt_attention: bad shape");
    CW_CHECK(isfinite(p->scale) && p->softcap >= 0.f && isfinite(p->softcap), CW_ERR_INVALID_ARG,
             "cw_prompt_attention: scale and softcap must be finite, softcap not negative");
    const uint64_t big = 1ull << 40;  // keeps the byte counts below from overflowing
    const size_t es = p->type == CW_GGUF_F32 ? 4 : 2, T = p->n_rows, L = p->n_keys,
                 D = p->head_dim, qw = p->n_heads * D, kw = p->n_kv * D;
    CW_CHECK(p->q_off < big && p->k_off < big && p->v_off < big && p->q_stride < (1ull << 30) &&
                 p->k_stride < (1ull << 30) && p->v_stride < (1ull << 30) &&
                 (p->q_stride >= qw || T == 1) &&
                 ((p->k_stride >= kw && p->v_stride >= kw) || L == 1),
             CW_ERR_INVALID_ARG, "cw_prompt_attention: bad offset or stride");
    BufEntry *q, *k, *v, *st, *ks = nullptr, *out;
    const size_t nq = ((T - 1) * p->q_stride + qw) * es, nk = ((L - 1) * p->k_stride + kw) * es,
                 nv = ((L - 1) * p->v_stride + kw) * es, no = T * qw * es,
                 ns = ((size_t)p->n_req + 1) * 4;
    CW_TRY(buf_get(ctx, p->q, &q, p->q_off * es + nq, "cw_prompt_attention(q)"));
    CW_TRY(buf_get(ctx, p->k, &k, p->k_off * es + nk, "cw_prompt_attention(k)"));
    CW_TRY(buf_get(ctx, p->v, &v, p->v_off * es + nv, "cw_prompt_attention(v)"));
    CW_TRY(buf_get(ctx, p->starts, &st, ns, "cw_prompt_attention(starts)"));
    if (p->key_starts)
        CW_TRY(buf_get(ctx, p->key_starts, &ks, ns, "cw_prompt_attention(key_starts)"));
    CW_TRY(buf_get(ctx, p->out, &out, no, "cw_prompt_attention(out)"));
    PromptArgs a{};
    a.q = (const char*)q->ptr + p->q_off * es;
    a.k = (const char*)k->ptr + p->k_off * es;
    a.v = (const char*)v->ptr + p->v_off * es;
    a.starts = (const int*)st->ptr;
    a.key_starts = ks ? (const int*)ks->ptr : nullptr;
    a.out = out->ptr;
    CW_CHECK(!spans_meet(a.out, no, a.q, nq) && !spans_meet(a.out, no, a.k, nk) &&
                 !spans_meet(a.out, no, a.v, nv) && !spans_meet(a.out, no, a.starts, ns) &&
                 !(ks && spans_meet(a.out, no, a.key_starts, ns)),
             CW_ERR_INVALID_ARG, "cw_prompt_attention: out lies on an input");
    a.q_stride = (long long)p->q_stride;
    a.k_stride = (long long)p->k_stride;
    a.v_stride = (long long)p->v_stride;
    a.n_req = (int)p->n_req;
    a.n_rows = (int)T;
    a.n_keys = (int)L;
    a.H = (int)p->n_heads;
    a.K = (int)p->n_kv;
    a.G = a.H / a.K;
    a.D = (int)D;
    // a window of all keys hides none; below that, sums with it stay in 32 bits although rows
    // before a request's first key count from a negative place
    a.window = p->window < L ? (int)p->window : 0;
    a.scale = p->scale != 0.f ? p->scale : 1.f / sqrtf((float)D);
    a.softcap = p->softcap;
    a.status = ctx->d_status;
    cudaSetDevice(ctx->device);
    OpScope scope(ctx, "prompt_attention");
    if (prompt_tc_takes(a, p->type)) {
        CW_TRY(prompt_tc_launch(ctx, a, p->type));
        if (p->type != CW_GGUF_F32) return CW_OK;  // else what the tensor cores left
    }
    if (p->type == CW_GGUF_F32) return prompt_dims<float>(ctx, a);
    if (p->type == CW_GGUF_F16) return prompt_dims<__half>(ctx, a);
    return prompt_dims<__nv_bfloat16>(ctx, a);
}
