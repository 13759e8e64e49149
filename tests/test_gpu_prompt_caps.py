"""Prompt attention with caps far above the scores: tanh is then nearly the identity, and a
difference of two numbers near the cap would lose the score."""
import numpy as np
import pytest

import prompt_ref
from test_gpu_prompt import make, run, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [2.0, 100.0, 256.0, 257.0, 1e4, 1e6, 1e20, 3e38])
@pytest.mark.parametrize("dtype,D", [("f32", 64), ("f32", 256), ("f16", 64), ("f16", 256), ("bf16", 128), ("f16", 36)])
def test_caps_of_every_size(ctx, dtype, D, cap):
    """A capped score is off by the score's own error and 2^-21 of itself; a cap of 256 at most
    may add 2^-22 of the cap (2^-14, an eighth of f16's rounding of the weight)."""
    c = make(np.random.default_rng(D), [200, 33], [200, 33], dtype, 4, 2, D)
    got = run(ctx, c, dtype, softcap=cap)
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, float(np.float32(cap)), D ** -0.5,
                                      c["q"])
    assert np.isfinite(got).all()
    extra = 2 * min(cap, 256.0) * 2.0 ** -22 * v if dtype != "f32" else 0.0
    assert np.abs(got - want).max() <= tolerance(dtype, s, v, 200) + extra
