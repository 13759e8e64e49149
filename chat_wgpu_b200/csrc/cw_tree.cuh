// cw_tree.cuh -- what the kernels of cw_tree_attention share: how the work is
// cut, what a row sees, and the partial states of a split key range.
//
// For one kv head a request with n nodes is a block of n * G query rows (G query
// heads per kv head, row = node * G + g) against its keys.  An ITEM is one kv head
// of one request and up to BM of its rows; a UNIT is one 64-key tile of an item.
// All units of the call, in request, kv head, row block, key order, are dealt to
// the CTAs in equal runs, so ragged requests, few requests and long contexts all
// fill the GPU alike.  The lengths are device data: every CTA sums the units of
// all requests (a few loads per thread) and finds its own run.  An item's start and end
// cost about as much as a few tiles and count as such: with tiles alone the CTAs with
// many short items ended a fifth later than the others.  An item cut by a
// run's end leaves one f32 partial state (maximum, sum, weighted values) per piece;
// a second launch joins the pieces in key order, so results do not depend on which
// CTA ran first.  (Joined by the last CTA to arrive instead, 150 us became 166: code
// that runs once comes from memory, and it took registers from the main loops.)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "cw_common.h"
#include "cw_device.cuh"

namespace cw {

constexpr int TR_TILE = 64;     // keys of a unit
constexpr int TR_NODES = 1024;  // most nodes of a request

struct TreePiece {  // an item whose first piece is this CTA's last one
    int row0, rows, head, block, count, slot;
};

struct TreeArgs {
    const void *q, *k, *v;
    void* out;
    const int *table, *lens, *starts, *positions;
    const uint32_t* mask;
    long long q_stride;
    int n_req, n_rows, max_nodes, words, H, K, G, D, page, n_pages, max_pages, window;
    float scale, softcap;
    int bm;            // rows of an item
    int pad;           // units that an item's start and end count as
    int dp;            // floats of a partial row
    float* part;       // [grid * 2][bm][dp]
    float2* ml;        // [grid * 2][bm] maximum (times log2 e) and sum
    TreePiece* pieces; // [grid]
    int* status;
};

struct TreeReq {
    int row0, n, len, keys, tile0, tiles, blocks;
};

__device__ __forceinline__ void tree_bad(const TreeArgs& a) {
    atomicCAS(a.status, DEV_OK, DEV_BAD_INPUT);
}

// First key that some row may see; pages before it need not be there.
__device__ __forceinline__ int tree_first(const TreeArgs& a, const TreeReq& q) {
    return a.window > 0 ? max(0, q.len - a.window + 1) : 0;
}
// Request r, every length clamped to the buffers; `report` notes a clamp.
__device__ __forceinline__ TreeReq tree_req(const TreeArgs& a, int r, bool report) {
    TreeReq q;
    const int s0 = a.starts[r], s1 = a.starts[r + 1], l = a.lens[r];
    q.row0 = min(max(s0, 0), a.n_rows);
    q.n = min(min(max(s1, q.row0), a.n_rows) - q.row0, a.max_nodes);
    const long long cap = (long long)a.max_pages * a.page;
    q.len = (int)min((long long)max(l, 0), cap);
    q.keys = (int)min((long long)q.len + q.n, cap);
    if (report && (s0 != q.row0 || s1 - s0 != q.n || l != q.len || q.keys != q.len + q.n))
        tree_bad(a);
    // a node's position is at least len: nothing before len - window + 1 is seen
    q.tile0 = min(tree_first(a, q), max(q.keys - 1, 0)) / TR_TILE;
    q.tiles = q.n > 0 ? (q.keys + TR_TILE - 1) / TR_TILE - q.tile0 : 0;
    q.blocks = (q.n * a.G + a.bm - 1) / a.bm;
    return q;
}
// Whether the page of the request's key j is in the cache.
__device__ __forceinline__ bool tree_has(const TreeArgs& a, int r, int j) {
    return (uint32_t)a.table[(size_t)r * a.max_pages + j / a.page] < (uint32_t)a.n_pages;
}
// Units of the request: its items' tiles, and `pad` more for each item's start and end.
__device__ __forceinline__ long long tree_units(const TreeArgs& a, const TreeReq& q) {
    return q.tiles ? (long long)a.K * q.blocks * (q.tiles + a.pad) : 0;
}

// This CTA's run of units, walked item by item: next is tile `pos` of item `item` of
// request r, whose lengths are q.
struct TreeRun {
    long long per;       // units of a CTA
    long long u;         // next unit, of all
    int r, item, pos;
    int left;            // units left in the run; above 0 there is a next tile
    TreeReq q;
};
struct TreeItem {
    TreeReq q;
    int r, head, block, rows;  // rows of this block
    int tile, tiles;           // tiles [tile, tile + tiles) of the item, from key tile q.tile0
    bool whole;
    long long first;           // the item's first unit, of all
};

// Past the end of an item, its padding and requests without tiles.
__device__ __forceinline__ void tree_advance(const TreeArgs& a, TreeRun& t) {
    if (t.pos < t.q.tiles) return;
    const int rest = t.q.tiles + a.pad - t.pos;
    t.u += rest;
    t.left -= rest;
    t.pos = 0;
    t.item++;
    while (t.left > 0 && t.item >= (t.q.tiles ? a.K * t.q.blocks : 0)) {
        t.q = tree_req(a, ++t.r, false);
        t.item = 0;
    }
}

// All threads (NT of them, a multiple of 32); sh is shared memory.
struct TreeShared {
    long long w[16], off;
    int r;
};
template <int NT>
__device__ TreeRun tree_run(const TreeArgs& a, TreeShared* sh) {
    long long* s_w = sh->w;
    long long& s_off = sh->off;
    int& s_r = sh->r;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool one = a.n_req <= NT;
    long long mine = 0;
    for (int r = tid; r < a.n_req; r += NT)
        mine += tree_units(a, tree_req(a, r, blockIdx.x == 0));
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(FULL, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) s_w[warp] = incl;
    if (tid == 0) s_r = 0, s_off = 0;
    __syncthreads();
    long long total = 0, before = 0;
    for (int w = 0; w < NT / 32; w++) {
        if (w == warp) before = total;
        total += s_w[w];
    }
    TreeRun t;
    t.per = max((total + gridDim.x - 1) / gridDim.x, 1ll);
    t.u = blockIdx.x * t.per;
    t.left = (int)max(0ll, min(t.per, total - t.u));
    if (t.left > 0) {
        if (one) {
            const long long e = before + incl - mine;
            if (mine > 0 && e <= t.u && t.u < e + mine) {
                s_r = tid;
                s_off = t.u - e;
            }
        } else {
            long long carry = 0;
            for (int b = 0; b < a.n_req; b += NT) {
                const int r = b + tid;
                const long long m = r < a.n_req ? tree_units(a, tree_req(a, r, false)) : 0;
                long long in = m;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long x = __shfl_up_sync(FULL, in, o);
                    if (lane >= o) in += x;
                }
                __syncthreads();
                if (lane == 31) s_w[warp] = in;
                __syncthreads();
                long long e = carry + in - m;
                for (int w = 0; w < warp; w++) e += s_w[w];
                if (m > 0 && e <= t.u && t.u < e + m) {
                    s_r = r;
                    s_off = t.u - e;
                }
                for (int w = 0; w < NT / 32; w++) carry += s_w[w];
            }
        }
    }
    __syncthreads();
    t.r = s_r;
    t.item = t.pos = 0;
    if (t.left > 0) {
        t.q = tree_req(a, t.r, false);
        t.item = (int)(s_off / (t.q.tiles + a.pad));
        t.pos = (int)(s_off - (long long)t.item * (t.q.tiles + a.pad));
        tree_advance(a, t);
    }
    return t;
}

// The next item of the run (t.left > 0).
__device__ __forceinline__ TreeItem tree_next(const TreeArgs& a, TreeRun& t) {
    TreeItem it;
    it.q = t.q;
    it.r = t.r;
    it.tile = t.pos;
    it.head = t.item / it.q.blocks;
    it.block = t.item - it.head * it.q.blocks;
    it.rows = min(a.bm, it.q.n * a.G - it.block * a.bm);
    it.tiles = min(it.q.tiles - it.tile, t.left);
    it.whole = it.tiles == it.q.tiles;
    it.first = t.u - it.tile;
    t.pos += it.tiles;
    t.u += it.tiles;
    t.left -= it.tiles;
    tree_advance(a, t);
    return it;
}

// Where an item's partial state goes: the run's first item in slot 0, a later one
// (it can only be the last) in slot 1.
__device__ __forceinline__ int tree_slot(const TreeRun& t, const TreeItem& it) {
    return it.first + it.tile == blockIdx.x * t.per ? 0 : 1;
}
// One thread, after the run's last item: what the joining launch finds.
__device__ __forceinline__ void tree_record(const TreeArgs& a, const TreeRun& t,
                                            const TreeItem& it, bool any) {
    TreePiece p = {};
    if (any && !it.whole && it.tile == 0) {
        p.row0 = it.q.row0;
        p.rows = it.rows;
        p.head = it.head;
        p.block = it.block;
        p.count = (int)((it.first + it.q.tiles - 1) / t.per - blockIdx.x) + 1;
        p.slot = tree_slot(t, it);
    }
    a.pieces[blockIdx.x] = p;
}

// Bit i: row m (node * G + g, of the whole request) sees key key0 + i.
__device__ __forceinline__ uint64_t tree_sees(const TreeArgs& a, const TreeReq& q, int m,
                                              int key0) {
    const int node = m / a.G;
    if (node >= q.n) return 0;
    const int row = q.row0 + node;
    const int live = min(q.keys - key0, 64);
    const uint64_t all = live <= 0 ? 0 : live == 64 ? ~0ull : (1ull << live) - 1;
    const int s = key0 - q.len;  // node index of key0
    uint64_t nodes = 0;          // bit i: sees node s + i
    const int s0 = max(s, 0);
    if (a.mask) {
        const uint32_t* w = a.mask + (size_t)row * a.words;
        const int w0 = s0 >> 5, sh = s0 & 31;
        const uint64_t x0 = w0 < a.words ? w[w0] : 0, x1 = w0 + 1 < a.words ? w[w0 + 1] : 0;
        const uint64_t x2 = w0 + 2 < a.words ? w[w0 + 2] : 0;
        nodes = (x0 | x1 << 32) >> sh;
        if (sh) nodes |= x2 << (64 - sh);
    } else {
        const int last = node - s0;  // sees nodes s0 .. node
        nodes = last < 0 ? 0 : last >= 63 ? ~0ull : (1ull << (last + 1)) - 1;
    }
    uint64_t prefix = 0;
    if (s < 0) {
        prefix = s <= -64 ? ~0ull : (1ull << -s) - 1;
        nodes = s <= -64 ? 0 : nodes << -s;
    }
    if (a.window > 0) {
        const long long pos = a.positions[row];
        const long long cut = pos - a.window + 1 - key0;  // keys before it are too old
        if (cut > 0) prefix = cut >= 64 ? 0 : prefix & (~0ull << cut);
        nodes &= all;
        if (pos - q.len >= a.window)  // else every node is near enough
            for (uint64_t left = nodes; left; left &= left - 1) {
                const int i = __ffsll((long long)left) - 1;
                if (pos - a.positions[q.row0 + s + i] >= a.window) nodes &= ~(1ull << i);
            }
    }
    return (prefix | nodes) & all;
}

// First key that row m's window still holds (0 without a window).
__device__ __forceinline__ int tree_edge(const TreeArgs& a, const TreeReq& q, int m) {
    const int node = m / a.G;
    if (a.window <= 0 || node >= q.n) return 0;
    return (int)max((long long)a.positions[q.row0 + node] - a.window + 1, 0ll);
}
// Whether rows may see the 64 keys from key0 differently; edge: the largest
// tree_edge of the rows.
__device__ __forceinline__ bool tree_partial(const TreeReq& q, int edge, int key0) {
    return key0 + TR_TILE > q.len || key0 < edge;
}

template <typename T> __device__ __forceinline__ float tree_f32(T x);
template <> __device__ __forceinline__ float tree_f32(float x) { return x; }
template <> __device__ __forceinline__ float tree_f32(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float tree_f32(__nv_bfloat16 x) {
    return __bfloat162float(x);
}
template <typename T> __device__ __forceinline__ T tree_to(float x);
template <> __device__ __forceinline__ float tree_to(float x) { return x; }
template <> __device__ __forceinline__ __half tree_to(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 tree_to(float x) {
    return __float2bfloat16_rn(x);
}

// Host side: the tcgen05 kernels of 16-bit caches.  tree_tc_takes
// says whether the call's shape is one of its own; a.bm, a.dp and the grid follow.
bool tree_tc_takes(const cw_tree_attn_args& p, const void* q, const void* k, const void* v);
int tree_tc_rows(const TreeArgs& a);
int tree_tc_grid(cw_ctx* ctx, const TreeArgs& a);
int tree_tc_launch(cw_ctx* ctx, const TreeArgs& a, uint32_t type, int grid);

}  // namespace cw
