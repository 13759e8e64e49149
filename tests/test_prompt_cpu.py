"""Host side of the prompt and logits operators, without a GPU: argument structs, refusals
of the C entry points and of the prepared calls, and the plain forms by hand."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import prompt_ref
from conftest import ROOT


def test_structs_match_the_header(tmp_path):
    from chat_wgpu_b200 import _lib
    pairs = {"cw_norm_rope_args": _lib.NormRopeArgs, "cw_prompt_attn_args": _lib.PromptAttnArgs,
             "cw_adjust_logits_args": _lib.AdjustLogitsArgs}
    body = "".join(
        f'printf("{n} sizeof %zu\\n", sizeof({n}));\n' + "".join(
            f'printf("{n} {f[0]} %zu\\n", offsetof({n}, {f[0]}));\n' for f in t._fields_)
        for n, t in pairs.items())
    src = tmp_path / "s.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "chatcuda.h"\nint main(void) {{\n{body}return 0; }}\n')
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, value = line.split()
        t = pairs[name]
        assert int(value) == (C.sizeof(t) if field == "sizeof" else getattr(t, field).offset), line


def test_null_arguments_are_refused():
    from chat_wgpu_b200 import _lib
    lib = _lib.load()
    for fn, t in (("cw_norm_rope", _lib.NormRopeArgs), ("cw_prompt_attention", _lib.PromptAttnArgs),
                  ("cw_adjust_logits", _lib.AdjustLogitsArgs)):
        assert getattr(lib, fn)(None, None) == 1, fn
        assert getattr(lib, fn)(None, C.byref(t())) == 1, fn
        assert b"bad arguments" in lib.cw_last_error()


def wrapped(t):
    from chat_wgpu_b200.context import Buffer
    return Buffer(None, 1, t)


def test_wrapped_tensors_of_another_type_or_layout_are_refused():
    import torch
    from chat_wgpu_b200.kernels.logits import AdjustLogits
    from chat_wgpu_b200.kernels.prompt import PromptAttention
    from chat_wgpu_b200.kernels.rope import NormRope
    i = lambda *s: wrapped(torch.zeros(*s, dtype=torch.int32))  # noqa: E731
    x = lambda *s: wrapped(torch.zeros(*s, dtype=torch.bfloat16))  # noqa: E731
    f = lambda *s: wrapped(torch.zeros(*s))  # noqa: E731
    rows = torch.zeros(5, 8 * 16, dtype=torch.bfloat16)
    q, k, v = (wrapped(t) for t in rows.split([64, 32, 32], dim=1))
    prompt = dict(q=q, k=k, v=v, starts=i(3), key_starts=i(3), out=x(5, 64), dtype="bf16", n_req=2, n_rows=5,
                  n_heads=4, n_kv=2, head_dim=16, n_keys=5, q_stride=128, k_stride=128, v_stride=128)
    with pytest.raises(ValueError, match="n_keys"):
        PromptAttention(None, **{**prompt, "n_keys": None})
    heads = dict(plan=i(4), positions=i(5), dtype="bf16", n_tokens=5, head_dim=16, eps=1e-6, n_heads=4, n_kv=2, q=q,
                 k=k, v=v, q_norm=f(16), k_norm=f(16), q_out=x(5, 64), k_out=x(5, 32), slots=i(5),
                 k_cache=x(1, 2, 16, 16), v_cache=x(1, 2, 16, 16), page_size=16, n_pages=1, q_stride=128, k_stride=128,
                 v_stride=128)
    logits = dict(logits=x(2, 40), out=x(2, 40), dtype="bf16", n_rows=2, vocab=40, penalties=f(2, 3), tokens=i(9),
                  starts=i(3), prompts=i(2), n_tokens=9, bias_tokens=i(3), bias_values=f(3), bias_starts=i(3), n_bias=3,
                  masks=i(1, 2), mask_rows=i(2), n_masks=1, best=i(2))
    for call, good, bad in (
            (PromptAttention, prompt, dict(q=f(5, 64), out=wrapped(torch.zeros(5, 128, dtype=torch.bfloat16)[:, ::2]),
                                           k_stride=32, starts=wrapped(torch.zeros(3, dtype=torch.int64)))),
            (NormRope, heads, dict(q_norm=x(16), k_norm=i(16), q_out=f(5, 64), v_stride=32, positions=f(5))),
            (AdjustLogits, logits, dict(penalties=i(2, 3), bias_values=x(3), tokens=f(9), out=f(2, 40), stride=48,
                                        best=wrapped(torch.zeros(2, dtype=torch.int64))))):
        call(None, **good)
        for name, value in bad.items():
            if name == "stride":
                wide = torch.zeros(2, 50, dtype=torch.bfloat16)[:, :40]
                with pytest.raises(ValueError, match="logits"):
                    call(None, **{**good, "logits": wrapped(wide), "stride": 48})
                call(None, **{**good, "logits": wrapped(wide), "stride": 50})
                continue
            with pytest.raises(ValueError, match=name.removesuffix("_stride")):
                call(None, **{**good, name: value})
        for number in (-1, 2 ** 32, 1.5):
            field = "n_rows" if "n_rows" in good else "n_tokens"
            with pytest.raises(ValueError, match=field):
                call(None, **{**good, field: number})


def test_plain_logits_by_hand():
    x = np.array([[1.0, -1.0, 2.0, 0.5]])
    got, best = prompt_ref.adjust(x, "f32", [[2.0, 0.25, 0.5]], [[0, 1, 2, 2]], [1], [[(3, 9.0), (3, 1.0)]],
                                  np.array([[True, True, False, True]]), [0])
    assert got.tolist() == [[0.5, -2.75, -np.inf, 1.5]] and best[0] == 3


def test_plain_attention_by_hand():
    """One head of one dim with equal scores: means of what each row sees."""
    v = np.arange(6.0).reshape(6, 1, 1)
    q = np.zeros((5, 1, 1))
    out, _, _ = prompt_ref.attention(q, v * 0, v, [0, 2, 5], [0, 4, 6], 2, 0.0, 1.0, q)
    # the last two of four keys' rows, a window of two; then three rows over two keys
    assert out.ravel().tolist() == [1.5, 2.5, 0.0, 4.0, 4.5]
