"""Prompt attention of f32 values of very different sizes: what a row does not see, or hardly
weighs, must not cost it bits."""
import numpy as np
import pytest

import prompt_ref
from test_gpu_prompt import make, run, tolerance

pytestmark = pytest.mark.gpu


def attention(c, D, window=0):
    return prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], window, 0.0, D ** -0.5, c["q"])


@pytest.mark.parametrize("big", [2.0 ** 13, 2.0 ** 20, 2.0 ** 30, 2.0 ** 40, 2.0 ** 59], ids=lambda x: f"2^{int(np.log2(x))}")
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("D", [40, 128])
def test_large_rows_out_of_sight(ctx, D, what, big):
    """A large key or value behind a row, or before its window, leaves it at f32 accuracy of
    what it does see."""
    c = make(np.random.default_rng(D), [400, 30], [400, 30], "f32", 4, 2, D)
    want, s, v = attention(c, D)
    c[what][350, 1] *= big
    got = run(ctx, c, "f32", same=True)
    unseen = np.ones(len(got), bool)
    unseen[350:400] = False
    assert np.abs(got - want)[unseen].max() <= tolerance("f32", s, v, 400)
    assert np.abs(got - want)[:, :2].max() <= tolerance("f32", s, v, 400)  # the other kv head
    # before the window of most rows
    c = make(np.random.default_rng(D), [400], [400], "f32", 4, 2, D)
    want, s, v = attention(c, D, 64)
    c[what][5, 0] *= big
    got = run(ctx, c, "f32", same=True, window=64)
    assert np.abs(got - want)[5 + 64:].max() <= tolerance("f32", s, v, 400)


def test_large_rows_in_sight(ctx):
    """A row whose own values are small beside the rest of its request's, pieces and many heads."""
    H, K, D = 8, 4, 64
    c = make(np.random.default_rng(3), [40, 12], [700, 300], "f32", H, K, D)
    size = np.exp2(np.random.default_rng(4).integers(-30, 30, (1000, K, 1)))
    c["v"] = (c["v"].astype(np.float32) * size.astype(np.float32)).astype(np.float64)
    got = run(ctx, c, "f32")
    want, s, _ = attention(c, D)
    # against the largest value that a row weighs: sum of w |v|, an f32 sum's own measure
    most = prompt_ref.attention(c["q"], c["k"], np.abs(c["v"]).max(-1, keepdims=True) + 0 * c["v"], c["starts"],
                                c["ks"], 0, 0.0, D ** -0.5, c["q"])[0]
    assert (np.abs(got - want) <= tolerance("f32", s, 1.0, 700) * most).all()


@pytest.mark.parametrize("down", [33, 36])
def test_light_keys_of_large_values(ctx, down):
    """A thousand keys of weights 2^-down of the largest, whose values are 2^12 of the heavy
    key's, count in the sum as f32 weights do.  A weight's score carries the score's error (2^-19
    of 25, twice) and its conversion less than 2^-11 of it: far below 2^-8 of the keys' share.
    Beside a result near 1 the f32 sums of a tile's 128 products and of ten tiles may drop a
    last place (2^-23) each."""
    H, K, D, n = 2, 1, 64, 1200
    c = make(np.random.default_rng(5), [16], [n], "f32", H, K, D)
    c["q"][:], c["k"][:], c["v"][:] = 0.0, 0.0, 4096.0
    c["q"][:, :, 0] = 8.0
    c["k"][:, 0, 0] = np.float32(-down * np.log(2.0))
    c["k"][300, 0, 0], c["v"][300] = 0.0, 1.0
    got = run(ctx, c, "f32")
    want, _, _ = attention(c, D)
    share = want - 1.0
    assert share.min() > 1e-5
    assert np.abs(got - want).max() <= 2.0 ** -8 * share.min() + 138 * 2.0 ** -23


@pytest.mark.parametrize("dims", [64, 100])
def test_rows_of_zeros(ctx, dims):
    """Rows of zeros among the keys and values, and queries of zeros, are exact whatever the
    others are."""
    c = make(np.random.default_rng(8), [260], [260], "f32", 4, 2, dims)
    c["k"][[0, 9, 200]] = 0.0
    c["v"][[3, 150]] = 0.0
    c["q"][[2, 100]] = 0.0
    got = run(ctx, c, "f32", same=True)
    want, s, v = attention(c, dims)
    assert np.abs(got - want).max() <= tolerance("f32", s, v, 260)
