"""Prompt attention in f32 where the dims of a row are of very different sizes: small ones keep
f32 accuracy of their own beside large ones."""
import numpy as np
import pytest

import prompt_ref
from test_gpu_prompt import make, run, tolerance

pytestmark = pytest.mark.gpu


def f32(x):
    return x.astype(np.float32).astype(np.float64)


@pytest.mark.parametrize("spread", [8, 20, 28])
@pytest.mark.parametrize("D,rows,keys", [(64, [300, 170], [300, 170]), (128, [40], [700]), (96, [12], [2600])])
def test_values_by_channel(ctx, D, rows, keys, spread):
    """Each dim of the result against the values of that dim, whatever the others' sizes."""
    rng = np.random.default_rng(spread)
    c = make(rng, rows, keys, "f32", 4, 2, D)
    c["v"] = f32(c["v"] * np.exp2(rng.integers(0, spread + 1, (1, 2, D)) - spread // 2))
    got = run(ctx, c, "f32")
    args = (c["starts"], c["ks"], 0, 0.0, D ** -0.5, c["q"])
    want, s, _ = prompt_ref.attention(c["q"], c["k"], c["v"], *args)
    most, _, _ = prompt_ref.attention(c["q"], c["k"], np.abs(c["v"]), *args)  # sum of w |v|, by dim
    assert (np.abs(got - want) <= tolerance("f32", s, 1.0, max(keys)) * most).all()


@pytest.mark.parametrize("spread", [8, 20, 28])
@pytest.mark.parametrize("D,rows,keys", [(64, [300, 170], [300, 170]), (128, [40], [700]), (96, [12], [2600])])
def test_scores_by_channel(ctx, D, rows, keys, spread):
    """Queries large where keys are small: each dim's product counts as in f32."""
    rng = np.random.default_rng(spread)
    c = make(rng, rows, keys, "f32", 4, 2, D)
    by = np.exp2(rng.integers(0, spread + 1, (1, 1, D)) - spread // 2)
    c["q"], c["k"] = f32(c["q"] * by), f32(c["k"] / by)
    got = run(ctx, c, "f32")
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, D ** -0.5, c["q"])
    assert np.abs(got - want).max() <= tolerance("f32", s, v, max(keys))


@pytest.mark.parametrize("large", ["q", "k"])
def test_channels_that_meet_zeros(ctx, large):
    """A channel of 2^28 that the other side has zeros in takes nothing from the scores."""
    D = 64
    c = make(np.random.default_rng(3), [300], [300], "f32", 4, 2, D)
    c["q"][:, :, 5] = c["k"][:, :, 5] = 0.0
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, D ** -0.5, c["q"])
    c[large][:, :, 5] = 2.0 ** 28
    got = run(ctx, c, "f32", same=True)
    # (the large channel's products are zeros, exactly)
    assert np.abs(got - want).max() <= tolerance("f32", s, v, 300)
