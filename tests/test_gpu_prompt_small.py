"""Prompt attention of f32 values far below one: they keep their bits, and keys that a row does
not see weigh nothing however small the scores."""
import numpy as np
import pytest

import prompt_ref
from test_gpu_prompt import make, run, tolerance

pytestmark = pytest.mark.gpu


def attention(c, D):
    return prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, D ** -0.5, c["q"])


@pytest.mark.parametrize("size", [2.0 ** -80, 2.0 ** -90, 2.0 ** -105, 2.0 ** -120], ids=lambda x: f"2^{int(np.log2(x))}")
def test_small_values(ctx, size):
    """Tiny values keep their bits, and tiny queries and keys weigh what they see alike."""
    D = 64
    c = make(np.random.default_rng(6), [300], [300], "f32", 4, 2, D)
    c["v"] = (c["v"] * size).astype(np.float32).astype(np.float64)
    got = run(ctx, c, "f32", same=True)
    want, s, v = attention(c, D)
    # below f32's normal range values are multiples of 2^-149
    assert np.abs(got - want).max() <= tolerance("f32", s, v, 300) + 300 * 2.0 ** -149
    for parts in ("qk", "q", "k"):
        c = make(np.random.default_rng(7), [300], [300], "f32", 4, 2, D)
        for p in parts:
            c[p] = (c[p] * size).astype(np.float32).astype(np.float64)
        got = run(ctx, c, "f32", same=True)
        want, s, v = attention(c, D)
        assert np.abs(got - want).max() <= tolerance("f32", s, v, 300), parts
