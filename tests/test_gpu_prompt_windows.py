"""Prompt attention of requests with fewer keys than rows, under windows of every size."""
import numpy as np
import pytest

import prompt_ref
from test_gpu_prompt import make, run, tolerance

pytestmark = pytest.mark.gpu

CASES = [  # dtype, heads, kv, dim, rows, keys
    ("f32", 4, 2, 64, [300, 40, 7], [290, 40, 250]),   # on pairs
    ("f32", 4, 2, 128, [200], [170]),
    ("f32", 4, 2, 256, [90, 20], [60, 30]),            # on the f32 kernel
    ("f32", 4, 2, 32, [20, 9], [3, 9]),
    ("f16", 4, 2, 64, [300, 40, 7], [290, 40, 250]),
    ("f16", 8, 4, 256, [150, 70], [20, 90]),
    ("bf16", 32, 8, 128, [200, 5, 64], [131, 0, 64]),
    ("bf16", 3, 1, 36, [50], [40]),                    # 16 bits on the f32 kernel
]


@pytest.mark.parametrize("window", [0, 7, 2 ** 31 - 1, 2 ** 31 - 60])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}x{c[2]}x{c[3]}-{c[4][0]}")
def test_fewer_keys_than_rows(ctx, case, window):
    """Rows before their request's first key give zeros, the others what they see."""
    dtype, H, K, D, rows, keys = case
    c = make(np.random.default_rng(sum(rows)), rows, keys, dtype, H, K, D, lead=2, gap=3)
    got = run(ctx, c, dtype, window=window)
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"].tolist(), c["ks"].tolist(), window, 0.0, D ** -0.5,
                                      np.full(c["q"].shape, 7.0))
    assert np.isfinite(got).all()
    for r, (n, m) in enumerate(zip(rows, keys)):
        first = c["starts"][r]
        assert (got[first:first + max(0, n - m)] == 0.0).all()
    assert np.abs(got - want).max() <= tolerance(dtype, s, v, max(keys))
    ctx.sync()


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("f32", 256), ("bf16", 128), ("f16", 256)])
@pytest.mark.parametrize("rows,keys", [([150, 30], [150, 30]), ([3], [2500])])
def test_windows_that_hide_nothing(ctx, dtype, D, rows, keys):
    """The bits of a window of all keys or more are those of none."""
    c = make(np.random.default_rng(D), rows, keys, dtype, 4, 2, D)
    plain = run(ctx, c, dtype)
    for window in (max(keys), max(keys) + 1, 2 ** 31 - 1):
        assert np.array_equal(run(ctx, c, dtype, window=window), plain), window
