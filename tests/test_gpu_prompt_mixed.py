"""Prompt attention of f32 batches that mix long requests with short and empty ones."""
import numpy as np
import pytest

import prompt_ref
from test_gpu_prompt import make, run, tolerance

pytestmark = pytest.mark.gpu

CASES = [  # heads, kv, dim, rows, keys (None: the rows)
    (4, 2, 64, [1100] + [1] * 30, None),
    (4, 2, 128, [0] * 31 + [1100] + [0] * 32, None),
    (4, 2, 40, [1, 159, 160, 161, 3, 700, 0, 127, 200], None),
    (2, 1, 64, [40, 3, 200, 1, 30], [159, 400, 300, 160, 30]),
    (2, 2, 64, [8, 1, 1, 30, 2], [1700, 100, 1900, 40, 30]),     # cut, with short ones between
    (4, 2, 64, [12] * 100, None),
    (2, 1, 32, [2, 1, 3] * 3, [500, 900, 300] * 3),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}-{len(c[3])}x{max(c[3])}")
def test_mixed_lengths(ctx, case):
    H, K, D, rows, keys = case
    c = make(np.random.default_rng(D + len(rows)), rows, keys or rows, "f32", H, K, D, lead=2, gap=3)
    got = run(ctx, c, "f32", same=keys is None)
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, D ** -0.5,
                                      np.full(c["q"].shape, 7.0))
    assert np.isfinite(got).all()
    assert np.abs(got - want).max() <= tolerance("f32", s, v, max(keys or rows))
    assert np.array_equal(got, run(ctx, c, "f32", same=keys is None))
    ctx.sync()


def test_short_requests_that_are_not_finite(ctx):
    """Short requests of NaN and infinities beside a long one keep them to themselves."""
    rows = [50, 400, 100, 700, 20]
    c = make(np.random.default_rng(2), rows, rows, "f32", 4, 2, 64)
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, 0.125, c["q"])
    for x, bad in zip("qkv", (np.nan, np.inf, -np.inf)):
        for r in (0, 2, 4):
            c[x][c["starts"][r]:c["starts"][r + 1]] = bad
    got = run(ctx, c, "f32", same=True)
    for r in (1, 3):
        at = slice(c["starts"][r], c["starts"][r + 1])
        assert np.abs(got[at] - want[at]).max() <= tolerance("f32", s, v, 700)
