"""cw_norm_rope refuses outputs that lie on an input other than the one they replace, before
anything is launched: the C entry point called without a GPU, on a context made by hand."""
import os
import subprocess

import pytest

from conftest import ROOT

CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
PROGRAM = r"""
#include <stdio.h>
#include "cw_common.h"

// 4 rows of two q heads, and of one kv head or two, of 8 elements
static cw_ctx ctx;
static char space[1 << 20];
static size_t used = 0;
static cw_buf at(char* p, size_t n) {
    cw::BufEntry e;
    e.ptr = p;
    e.nbytes = n;
    cw_buf id = ctx.next_id++;
    ctx.bufs[id] = e;
    return id;
}
static cw_buf make(size_t floats) {
    cw_buf b = at(space + used, floats * 4);
    used += (floats * 4 + 255) / 256 * 256;
    return b;
}
int main(void) {
    const int T = 4, H = 2, D = 8;
    ctx.sm_count = 148;
    int bad = 0;
    for (int kv = 1; kv <= 2; kv++) {
        const int K = kv;
        cw_norm_rope_args a = {};
        a.plan = make(D);
        ctx.bufs[a.plan].rope_dim = D;
        a.positions = make(T);
        a.slots = make(T);
        a.q = make(T * H * D);
        a.k = make(T * K * D);
        a.v = make(T * K * D);
        a.q_out = make(T * H * D);
        a.k_out = make(T * K * D);
        a.k_cache = make(2 * K * 16 * D);
        a.v_cache = make(2 * K * 16 * D);
        a.q_norm = make(D);
        a.k_norm = make(D);
        a.q_stride = H * D;
        a.k_stride = a.v_stride = K * D;
        a.n_tokens = T;
        a.n_heads = H;
        a.n_kv = K;
        a.head_dim = D;
        a.page_size = 16;
        a.n_pages = 2;
        // refused: 1 (an argument).  Past the checks the launch fails for want of a device.
        auto expect = [&](const char* what, cw_norm_rope_args x, bool refused) {
            const int rc = cw_norm_rope(&ctx, &x);
            const bool ok = refused ? rc == CW_ERR_INVALID_ARG : rc != CW_OK && rc != CW_ERR_INVALID_ARG;
            if (!ok) printf("kv %d: %s: %d %s\n", kv, what, rc, cw_last_error());
            bad += !ok;
        };
        cw_norm_rope_args x = a;
        expect("apart", x, false);
        x.q_out = x.q, x.k_out = x.k;
        expect("in place", x, false);
        x.v = x.k;
        expect("k in place, v the same rows", x, true);
        x.k_out = a.k_out;
        expect("v the same rows as k", x, false);
        x = a, x.k_out = a.k, x.v = at((char*)ctx.bufs[a.k].ptr, ctx.bufs[a.k].nbytes);
        expect("k in place, v the same rows by another handle", x, true);
        if (H == K) {
            x = a, x.k = a.q, x.q_out = a.q;
            expect("q in place, k the same rows", x, true);
            x = a, x.v = a.q, x.q_out = a.q;
            expect("q in place, v the same rows", x, true);
            x = a, x.k = a.q, x.k_out = a.q;
            expect("k in place, q the same rows", x, true);
            x = a, x.k = a.q;
            expect("k the same rows as q", x, false);
        }
        x = a, x.k_norm = at((char*)ctx.bufs[a.q].ptr, D * 4), x.q_out = a.q;
        expect("q in place, weights in its rows", x, true);
        x = a, x.slots = a.q, x.q_out = a.q;
        expect("q in place, slots in its rows", x, true);
    }
    return bad;
}
"""


def test_outputs_on_other_inputs_are_refused(tmp_path):
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: without a GPU only")
    from chat_wgpu_b200 import _lib
    src, exe = tmp_path / "o.cpp", str(tmp_path / "o")
    src.write_text(PROGRAM)
    lib = os.path.dirname(_lib.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(lib, "csrc"), "-I", os.path.join(ROOT, "include"), "-I",
                    f"{CUDA}/include", str(src), "-o", exe, _lib.LIB_PATH, f"-Wl,-rpath,{lib}", f"-L{CUDA}/lib64",
                    "-lcudart"], check=True)
    out = subprocess.run([exe], capture_output=True, text=True,
                         env={**os.environ, "LD_LIBRARY_PATH": f"{CUDA}/lib64"})
    assert out.returncode == 0, out.stdout + out.stderr
