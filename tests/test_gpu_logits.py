"""Penalties, biases and masks on logits on the device against their definition, bit for bit."""
import numpy as np
import pytest

import paged_ref as ref
import prompt_ref

pytestmark = pytest.mark.gpu


def i32(ctx, a):
    return ctx.storage_u32(np.ascontiguousarray(a, np.int32).view(np.uint32))


def flat(lists, lead=0):
    starts = lead + np.concatenate([[0], np.cumsum([len(x) for x in lists])])
    return starts, [y for x in lists for y in x]


def run(ctx, x, dtype, penalties=None, lists=None, prompts=None, biases=None, masks=None, mask_rows=None,
        pad=0, off=0, in_place=False, lead=0, best=True, bad=False):
    from chat_wgpu_b200 import CwError
    from chat_wgpu_b200.kernels.logits import AdjustLogits
    n, V = x.shape
    rows = np.full((n, V + pad), 1e4)
    rows[:, :V] = x
    src = ref.upload(ctx, np.concatenate([np.full(off, 3.0), rows.ravel()]), dtype)
    out = src if in_place else ref.upload(ctx, np.zeros((n, V)), dtype)
    more = {}
    if penalties is not None:
        starts, tokens = flat(lists, lead)
        tokens = [V + 5] * lead + tokens  # before the first list: nobody's
        more.update(penalties=ctx.storage(penalties), starts=i32(ctx, starts), n_tokens=len(tokens),
                    tokens=i32(ctx, tokens or [0]), prompts=None if prompts is None else i32(ctx, prompts))
    if biases is not None:
        starts, pairs = flat(biases)
        more.update(bias_starts=i32(ctx, starts), bias_tokens=i32(ctx, [p[0] for p in pairs] or [0]),
                    bias_values=ctx.storage([p[1] for p in pairs] or [0.0]), n_bias=len(pairs))
    if masks is not None:
        bits = np.zeros((len(masks), -(-V // 32) * 32), np.uint8)
        bits[:, :V] = masks
        more.update(masks=ctx.storage_u32(np.packbits(bits, axis=1, bitorder="little").view(np.uint32)),
                    n_masks=len(masks), mask_rows=None if mask_rows is None else i32(ctx, mask_rows))
    top = i32(ctx, np.full(n, -1))
    AdjustLogits(ctx, logits=src, out=out, dtype=dtype, n_rows=n, vocab=V, off=off, stride=V + pad,
                 best=top if best else None, **more)()
    if bad:
        with pytest.raises(CwError) as e:
            ctx.sync()
        assert e.value.status == 1
    got = ref.read(ctx, out, dtype, (n, V))
    return got, ctx.read_u32(top, n).astype(np.int64)


CASES = [  # dtype, rows, vocab, history, biases, masks, pad, off
    ("f32", 1, 1, 3, 1, 0, 0, 0),
    ("f32", 1, 151936, 300, 5, 0, 0, 0),
    ("f32", 8, 256000, 1000, 0, 3, 0, 0),
    ("f32", 3, 32003, 500, 40, 2, 0, 0),
    ("f32", 5, 1000, 200, 30, 2, 24, 3),
    ("f32", 2, 777, 50, 3, 1, 3, 0),
    ("f16", 4, 32003, 500, 40, 2, 5, 1),
    ("f16", 7, 4096, 5000, 300, 4, 8, 8),
    ("f16", 300, 100, 20, 5, 6, 0, 0),
    ("bf16", 16, 151936, 2000, 40, 5, 0, 0),
    ("bf16", 3, 49999, 100, 1000, 1, 1, 0),
    ("bf16", 9, 33, 70, 20, 3, 7, 9),
    ("bf16", 2, 900001, 3000, 300, 2, 7, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_adjust_logits(ctx, case):
    dtype, n, V, history, bias, masks, pad, off = case
    rng = np.random.default_rng(n + V)
    x = ref.rounded(rng.normal(0, 4, (n, V)), dtype)
    lists = [(V * rng.random(rng.integers(0, history + 1)) ** 3).astype(int).tolist() for _ in range(n)]
    lists[-1] = lists[-1] + [V - 1, 0, V - 1]
    prompts = [int(rng.integers(-1, len(t) + 2)) for t in lists]
    lead = [min(max(p, 0), len(t)) for p, t in zip(prompts, lists)]
    pen = np.stack([rng.choice([1.0, 1.1, 1.3], n), rng.choice([0.0, 0.1, 0.7], n),
                    rng.choice([0.0, 0.2, -0.3], n)], 1).astype(np.float32)
    pen[0] = 1.2, 0.1, 0.3
    biases = [[(int(rng.integers(0, V)), float(np.float32(rng.normal(0, 5)))) for _ in range(rng.integers(0, bias + 1))]
              for _ in range(n)]
    allow = rng.random((max(masks, 1), V)) < 0.5
    rows = rng.integers(-1, masks, n) if masks else None
    want, top = prompt_ref.adjust(x, dtype, pen, lists, lead, biases, allow if masks else None, rows)
    got, best = run(ctx, x, dtype, pen, lists, prompts, biases, allow if masks else None, rows, pad, off)
    assert np.array_equal(got, want) and np.array_equal(best, top)
    ctx.sync()
    # each part by itself, and in place
    if pad == off == 0:
        want, top = prompt_ref.adjust(x, dtype, pen, lists)
        got, best = run(ctx, x, dtype, pen, lists, in_place=True)
        assert np.array_equal(got, want) and np.array_equal(best, top)
        want, top = prompt_ref.adjust(x, dtype, biases=biases)
        got, best = run(ctx, x, dtype, biases=biases)
        assert np.array_equal(got, want) and np.array_equal(best, top)
        if masks:
            want, top = prompt_ref.adjust(x, dtype, masks=allow, mask_rows=rows)
            got, _ = run(ctx, x, dtype, masks=allow, mask_rows=rows, best=False)
            assert np.array_equal(got, want)
    got, best = run(ctx, x, dtype)
    want, top = prompt_ref.adjust(x, dtype)
    assert np.array_equal(got, want) and np.array_equal(best, top)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_adjust_logits_special_values(ctx, dtype):
    """Masked NaN and infinities go, seen ones stay; nothing allowed: index 0; ties and the
    type's lowest value: the lowest index."""
    V = 5000
    rng = np.random.default_rng(2)
    x = ref.rounded(rng.normal(0, 1, (6, V)), dtype)
    x[0, 10], x[0, 20], x[0, 4000] = np.nan, np.inf, np.inf
    x[1, 10], x[1, 20], x[1, 30] = np.nan, np.inf, -np.inf
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895313892515355e38}[dtype]
    x[3] = low
    x[4] = 2.5
    x[5, 77:4990] = 100.0
    masks = np.ones((6, V), bool)
    masks[1, [10, 20]] = False
    masks[2] = False
    masks[4, :4321] = False
    want, top = prompt_ref.adjust(x, dtype, masks=masks)
    got, best = run(ctx, x, dtype, masks=masks)
    assert np.array_equal(got, want, equal_nan=True) and np.array_equal(best, top)
    assert best[0] == 20 and best[2] == 0 and best[3] == 0 and best[4] == 4321 and best[5] == 77
    assert (got[2] == -np.inf).all()


def test_adjust_logits_repeated_entries(ctx):
    """The last bias of a token holds, however long the list; counts add up; penalties of
    one and zero leave even a NaN-free history unread."""
    V = 300
    x = np.zeros((2, V), np.float32)
    biases = [[(7, 1.0)] * 4000 + [(7, 2.5), (8, 1.0), (7, -3.0)], []]
    lists = [[5] * 70000 + [6] * 3, [V + 9, -4, 2 ** 31 - 1]]
    pen = np.array([[2.0, 0.5, 0.25], [1.0, 0.0, 0.0]], np.float32)
    got, best = run(ctx, x, "f32", pen, lists, biases=biases)
    assert got[0, 7] == -3.0 and got[0, 8] == 1.0 and got[0, 5] == -35000.25 and got[0, 6] == -1.75
    assert best[0] == 8 and best[1] == 0 and not got[1].any()
    ctx.sync()


def test_adjust_logits_bad_values(ctx):
    """Tokens outside the vocabulary, lists that pass their buffer and mask rows past the
    masks are skipped and reported."""
    from chat_wgpu_b200 import CwError
    V = 100
    x = np.ones((2, V), np.float32)
    pen = np.array([[2.0, 0.0, 0.0]] * 2, np.float32)

    def reported(want, *args, **more):
        got, _ = run(ctx, x, "f32", *args, bad=True, **more)
        assert np.array_equal(got, want)

    want, _ = prompt_ref.adjust(x, "f32", pen, [[3], [4]])
    reported(want, pen, [[3, V, -1], [4, 2 ** 30]])
    want, _ = prompt_ref.adjust(x, "f32", biases=[[(3, 1.0)], []])
    reported(want, biases=[[(3, 1.0), (V, 2.0)], [(-7, 1.0)]])
    masks = np.zeros((1, V), bool)
    reported(np.stack([np.full(V, -np.inf), x[1]]), masks=masks, mask_rows=[0, 1])
    # a list that ends behind the buffer
    from chat_wgpu_b200.kernels.logits import AdjustLogits
    out = ctx.storage(np.zeros(2 * V))
    AdjustLogits(ctx, logits=ctx.storage(x), out=out, dtype="f32", n_rows=2, vocab=V, penalties=ctx.storage(pen),
                 tokens=i32(ctx, [3, 4]), starts=i32(ctx, [0, 1, 2 ** 31 - 1]), n_tokens=2)()
    with pytest.raises(CwError):
        ctx.sync()
    want, _ = prompt_ref.adjust(x, "f32", pen, [[3], [4]])
    assert np.array_equal(ctx.read(out, 2 * V).reshape(2, V), want)


def test_adjust_logits_refusals(ctx):
    from chat_wgpu_b200 import CwError
    from chat_wgpu_b200.kernels.logits import AdjustLogits
    b = lambda n: ctx.storage(np.zeros(n))  # noqa: E731
    x, o, best, pen, st, tok = b(64), b(64), b(4), b(12), b(5), b(8)
    good = dict(logits=x, out=o, dtype="f32", n_rows=4, vocab=16, best=best, penalties=pen, tokens=tok, starts=st,
                prompts=b(4), n_tokens=8, bias_tokens=b(3), bias_values=b(3), bias_starts=b(5), n_bias=3, masks=b(2),
                mask_rows=b(4), n_masks=2)
    AdjustLogits(ctx, **good)()
    ctx.sync()
    for bad in (dict(n_rows=0), dict(n_rows=5), dict(n_rows=65536), dict(vocab=0), dict(vocab=17), dict(off=1),
                dict(stride=15), dict(stride=17), dict(logits=None), dict(out=None), dict(best=b(3)),
                dict(penalties=b(11)), dict(starts=None), dict(starts=b(4)), dict(tokens=b(7)), dict(prompts=b(3)),
                dict(bias_tokens=None), dict(bias_values=b(2)), dict(bias_starts=b(4)), dict(masks=b(1)),
                dict(n_masks=0), dict(mask_rows=None), dict(mask_rows=b(3)), dict(best=x), dict(best=o), dict(out=pen),
                dict(best=st), dict(off=8, n_rows=3, out=x)):
        with pytest.raises(CwError) as e:
            AdjustLogits(ctx, **{**good, **bad})()
        assert e.value.status == 1, bad
