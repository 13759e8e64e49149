"""Host side of the paged operators, without a GPU: argument structs, refusals of the C
entry points, the plain page plan, and the drafts of the tree decode."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import paged_ref as ref
from conftest import ROOT


def test_structs_match_the_header(tmp_path):
    """Every field of the ctypes structs sits where the C compiler puts it."""
    from chat_wgpu_b200 import _lib
    pairs = {"cw_page_plan_args": _lib.PagePlanArgs, "cw_rope_scaling": _lib.RopeScaling,
             "cw_rope_append_args": _lib.RopeAppendArgs, "cw_tree_attn_args": _lib.TreeAttnArgs}
    body = "".join(
        f'printf("{n} sizeof %zu\\n", sizeof({n}));\n' + "".join(
            f'printf("{n} {f[0]} %zu\\n", offsetof({n}, {f[0]}));\n' for f in t._fields_)
        for n, t in pairs.items())
    src = tmp_path / "s.c"
    src.write_text(f'#include <stdio.h>\n#include "chatcuda.h"\nint main(void) {{\n{body}return 0; }}\n')
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, value = line.split()
        t = pairs[name]
        assert int(value) == (C.sizeof(t) if field == "sizeof" else getattr(t, field).offset), line


def test_null_arguments_are_refused():
    from chat_wgpu_b200 import _lib
    lib = _lib.load()
    for fn, t in (("cw_page_plan", _lib.PagePlanArgs), ("cw_rope_append", _lib.RopeAppendArgs),
                  ("cw_tree_attention", _lib.TreeAttnArgs)):
        assert getattr(lib, fn)(None, None) == 1, fn
        assert getattr(lib, fn)(None, C.byref(t())) == 1, fn
        assert b"bad arguments" in lib.cw_last_error()
    assert lib.cw_rope_plan(None, 16, 1e4, None, None) == 1
    assert lib.cw_buf_wrap(None, None, 0, None) == 1
    assert lib.cw_ctx_create_on_stream(0, None, None) == 1


def test_python_calls_refuse_unknown_names():
    from chat_wgpu_b200.kernels._util import type_code
    assert [type_code(t) for t in ("f32", "f16", "bf16")] == [0, 1, 30]
    with pytest.raises(ValueError):
        type_code("f64")


def test_plain_plan_by_hand():
    """Three requests: a page begun, none, one full; two free pages for three wanted."""
    table = np.array([[7, -1], [-1, -1], [9, -1]], np.int32)
    p = ref.plan([3, 0, 4], [2, 4, 1], [5, 6], table, 4, 9)
    assert p["used"] == 3 and list(p["starts"]) == [0, 2, 6, 7]
    assert p["table"].tolist() == [[7, 5], [6, -1], [9, -1]]
    assert list(p["slots"]) == [31, 20, 24, 25, 26, 27, -1, -1, -1]
    assert list(p["positions"]) == [3, 4, 0, 1, 2, 3, 4, 0, 0]
    assert list(p["owners"]) == [0, 0, 1, 1, 1, 1, 2, -1, -1]


def test_drafts_are_trees():
    from chat_wgpu_b200.treedecode import lookup_draft
    assert lookup_draft([1, 2, 3]) == []
    nodes = lookup_draft([1, 2, 3, 4, 1, 2, 3, 5, 1, 2], width=2, depth=3, match=2)
    # ... 3, 5, 1 and ... 3, 4, 1 share their first token
    assert nodes == [(-1, 3), (0, 5), (1, 1), (0, 4), (3, 1)]
    assert all(p < i for i, (p, _) in enumerate(nodes))
