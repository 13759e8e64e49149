"""Causal attention of packed prompts on the device against the 64-bit form."""
import numpy as np
import pytest

import paged_ref as ref
import prompt_ref

pytestmark = pytest.mark.gpu


def i32(ctx, a):
    return ctx.storage_u32(np.ascontiguousarray(a, np.int32).view(np.uint32))


def tolerance(dtype, big_s, big_v, keys):
    """A score's terms carry at most 2^-21 each and its f32 sum as much, so a score is off by
    2^-19 of the sum of its terms' magnitudes and weights by twice that; the exponential, the
    running rescales and the sums over the keys 2^-18 (2^-24 times the tiles' additions);
    a 16-bit type rounds each weight once (u) and the result once (u).  All on values of at
    most big_v.  f16 weights below 2^-24 of the largest possible are lost: 2^-31 a key."""
    u = 0.0 if dtype == "f32" else ref.UNIT[dtype]
    lost = keys * 2.0 ** -31 if dtype == "f16" else 0.0
    return big_v * (2 * 2.0 ** -19 * big_s + 2.0 ** -18 + 2 * u + lost)


def make(rng, rows, keys, dtype, H, K, D, lead=0, gap=0, q_size=2.0):
    """Packed requests with `lead` rows and keys before the first and `gap` after the last,
    which hold NaN and belong to nobody."""
    starts = lead + np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    ks = lead + np.concatenate([[0], np.cumsum(keys)]).astype(np.int32)
    T, L = int(starts[-1]) + gap, int(ks[-1]) + gap
    q = ref.rounded(rng.normal(0, q_size, (T, H, D)), dtype)
    k, v = (ref.rounded(rng.normal(0, 1, (L, K, D)), dtype) for _ in range(2))
    for x, s in ((q, starts), (k, ks), (v, ks)):
        x[:s[0]] = np.nan
        x[s[-1]:] = np.nan
    return dict(q=q, k=k, v=v, starts=starts, ks=ks)


def run(ctx, c, dtype, window=0, softcap=0.0, scale=0.0, same=False, pad=0, off=0, bad=False):
    from chat_wgpu_b200 import CwError
    from chat_wgpu_b200.kernels.prompt import PromptAttention
    (T, H, D), (L, K, _) = c["q"].shape, c["k"].shape

    def rows(x):
        y = np.full((len(x), x[0].size + pad), np.nan)
        y[:, off:off + x[0].size] = x.reshape(len(x), -1)
        return ref.upload(ctx, y, dtype)

    o = ref.upload(ctx, np.full((T, H, D), 7.0), dtype)
    PromptAttention(ctx, q=rows(c["q"]), k=rows(c["k"]), v=rows(c["v"]), starts=i32(ctx, c["starts"]),
                    key_starts=None if same else i32(ctx, c["ks"]), out=o, dtype=dtype,
                    n_req=len(c["starts"]) - 1, n_rows=T, n_keys=L, n_heads=H, n_kv=K, head_dim=D,
                    window=window, softcap=softcap, scale=scale, q_off=off, k_off=off, v_off=off,
                    q_stride=H * D + pad, k_stride=K * D + pad, v_stride=K * D + pad)()
    if bad:
        with pytest.raises(CwError) as e:
            ctx.sync()
        assert e.value.status == 1
    return ref.read(ctx, o, dtype, (T, H, D))


CASES = [  # dtype, heads, kv, dim, rows, keys (None: the rows), options
    ("f32", 2, 1, 16, [1], None, {}),
    ("f32", 16, 8, 128, [17], None, {}),
    ("f32", 4, 2, 64, [1, 0, 63, 64, 65, 127, 1, 130], None, {}),
    ("f32", 7, 7, 33, [40, 9], None, dict(window=5)),
    ("f32", 8, 4, 256, [90, 30], None, dict(window=50, softcap=20.0)),
    ("f32", 6, 2, 48, [5, 30, 7], [100, 30, 3], {}),
    ("f32", 8, 1, 80, [70], [200], dict(window=64)),
    ("f32", 4, 4, 3, [33], None, dict(pad=3, off=1)),
    ("f32", 16, 8, 128, [300, 129], [300, 400], {}),
    ("f16", 4, 2, 64, [1, 0, 63, 64, 65, 127, 1, 130], None, {}),
    ("f16", 8, 4, 256, [150, 70], None, dict(window=60, softcap=50.0)),
    ("f16", 8, 4, 256, [129, 64, 1], [300, 64, 140], {}),
    ("f16", 12, 4, 96, [77, 200], None, dict(softcap=10.0)),
    ("f16", 4, 2, 36, [100], None, {}),
    ("f16", 3, 1, 128, [61, 90], None, dict(pad=3, off=1)),
    ("f16", 14, 2, 64, [100, 37], None, {}),
    ("bf16", 32, 8, 128, [130, 64, 1, 200], None, {}),
    ("bf16", 32, 8, 128, [300], None, dict(window=90)),
    ("bf16", 32, 8, 128, [40, 7, 33], [400, 135, 33], {}),
    ("bf16", 8, 8, 128, [520, 129], None, {}),
    ("bf16", 8, 8, 48, [250, 10], None, dict(window=128)),
    ("bf16", 16, 2, 64, [260], None, {}),
    ("bf16", 24, 8, 80, [333], None, {}),
    ("bf16", 1, 1, 8, [9, 2, 3], None, {}),
    ("bf16", 7, 1, 128, [257], [300], {}),
    ("bf16", 12, 1, 192, [90], None, {}),
    ("bf16", 64, 1, 64, [40, 5], None, {}),
    ("f16", 130, 1, 64, [7], None, {}),
    ("bf16", 4, 2, 200, [140], [150], dict(window=33)),
    # few rows over many keys, which are cut and joined
    ("bf16", 32, 8, 128, [1], [3000], {}),
    ("bf16", 32, 8, 128, [3, 0, 40, 1], [2100, 5, 1300, 2], {}),
    ("f16", 8, 4, 256, [5, 70], [2000, 1500], dict(window=700, softcap=20.0)),
    ("f16", 14, 2, 64, [19], [1700], {}),
    ("f32", 16, 8, 128, [3], [2500], {}),
    ("f32", 16, 8, 128, [9], [2500], {}),
    ("f32", 16, 8, 40, [90, 7], [1200, 1900], dict(softcap=15.0)),
    ("f32", 8, 4, 256, [2, 9], [1800, 900], {}),
    ("f32", 2, 2, 130, [4], [1400], dict(window=600, pad=3, off=1)),
    ("bf16", 3, 1, 128, [40], [1500], dict(pad=3, off=1)),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}x{c[2]}x{c[3]}-{max(c[4])}x{len(c[4])}")
def test_prompt_attention(ctx, case):
    dtype, H, K, D, rows, keys, opt = case
    opt = dict(dict(pad=24, off=8), **opt)
    rng = np.random.default_rng(sum(rows) + D)
    c = make(rng, rows, keys or rows, dtype, H, K, D, lead=3, gap=5)
    got = run(ctx, c, dtype, same=keys is None, **opt)
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], opt.get("window", 0),
                                      opt.get("softcap", 0.0), D ** -0.5, np.full(c["q"].shape, 7.0))
    assert np.isfinite(got).all()
    mine = np.zeros(len(got), bool)
    mine[c["starts"][0]:c["starts"][-1]] = True
    assert (got[~mine] == 7.0).all()
    assert np.abs(got - want).max() <= tolerance(dtype, s, v, max(keys or rows))
    ctx.sync()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_prompt_scale_and_bits(ctx, dtype):
    """A given scale, rows side by side; the bits of two runs are the same."""
    c = make(np.random.default_rng(5), [150, 37], [150, 37], dtype, 8, 2, 64)
    got = run(ctx, c, dtype, scale=0.3, same=True)
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, 0.3, c["q"])
    assert np.abs(got - want).max() <= tolerance(dtype, s, v, 150)
    assert np.array_equal(got, run(ctx, c, dtype, scale=0.3, same=True))


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("f16", 64), ("bf16", 128), ("f16", 256)])
def test_prompt_not_finite(ctx, dtype, D):
    """Keys and values that are not finite reach the rows that see them and no others."""
    H, K = 4, 2
    c = make(np.random.default_rng(6), [200, 150], [200, 150], dtype, H, K, D)
    clean, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, D ** -0.5, c["q"])
    c["v"][170, 1, 3] = np.inf
    c["v"][190, 1, 5] = np.nan
    c["k"][198, 0, 2] = np.nan
    c["v"][200 + 149, 0, 0] = -np.inf
    got = run(ctx, c, dtype, same=True)
    tol = tolerance(dtype, s, v, 200)
    assert np.isnan(got[198:200, :2]).all()
    assert (got[170:200, 2:, 3] == np.inf).all() and np.isnan(got[190:200, 2:, 5]).all()
    assert (got[349, :2, 0] == -np.inf).all()
    bad = np.zeros(got.shape, bool)
    bad[198:200, :2] = bad[170:200, 2:, 3] = bad[190:200, 2:, 5] = bad[349, :2, 0] = True
    assert np.abs(got[~bad] - clean[~bad]).max() <= tol


@pytest.mark.parametrize("dtype,D", [("f32", 128), ("f32", 200), ("f16", 256), ("bf16", 64)])
def test_prompt_pieces_not_finite(ctx, dtype, D):
    """Cut items: what is not finite reaches the rows that see it, whichever piece it is in; a
    piece whose keys all score -inf keeps the NaN of 0 times an infinite value."""
    H, K = 2, 1
    c = make(np.random.default_rng(8), [4], [2600], dtype, H, K, D)
    c["q"][:, :, 0] = 1.0
    c["k"][:900, :, 0] = -np.inf
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, D ** -0.5, c["q"])
    c["v"][300, 0, 5] = np.inf     # weighs nothing: NaN
    c["v"][1500, 0, 9] = np.inf    # weighs something
    c["v"][2599, 0, 1] = np.nan    # the last row alone sees it
    c["k"][2598, 0, 2] = np.nan    # the last two rows see it
    got = run(ctx, c, dtype)
    assert np.isnan(got[:, :, 5]).all() and (got[:2, :, 9] == np.inf).all() and np.isnan(got[2:]).all()
    rest = np.setdiff1d(np.arange(D), [5, 9])
    assert np.abs(got[:2][:, :, rest] - want[:2][:, :, rest]).max() <= tolerance(dtype, s, v, 2600)


@pytest.mark.parametrize("keys", [300, 2600])
def test_prompt_repeated(ctx, keys):
    """Calls on the same rows give the same bits: an item's end waits for its last product."""
    c = make(np.random.default_rng(9), [4, 70], [keys, keys - 40], "f16", 2, 1, 256)
    first = run(ctx, c, "f16")
    for _ in range(40):
        assert np.array_equal(run(ctx, c, "f16"), first)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_prompt_scores_of_minus_infinity(ctx, dtype):
    """Keys that score -inf weigh nothing, in the first tile and in a later one; a row that
    sees no other gives zeros."""
    H, K, D = 2, 1, 64
    c = make(np.random.default_rng(7), [300], [300], dtype, H, K, D)
    c["q"][:, :, 0] = 1.0
    dead = np.r_[0:140, 210:230]
    c["k"][dead, :, 0] = -np.inf
    got = run(ctx, c, dtype, same=True)
    assert (got[:140] == 0).all()
    k, v = c["k"].copy(), c["v"]
    want = np.zeros_like(got)
    live = np.setdiff1d(np.arange(300), dead)
    big = 0.0
    for t in range(140, 300):
        j = live[live <= t]
        for h in range(H):
            sc = k[j, 0] @ c["q"][t, h] / 8
            w = np.exp(sc - sc.max())
            want[t, h] = w @ v[j, 0] / w.sum()
            big = max(big, (np.abs(k[j, 0]) @ np.abs(c["q"][t, h])).max() / 8)
    assert np.abs(got - want).max() <= tolerance(dtype, big, np.abs(v).max(), 300)


@pytest.mark.parametrize("dtype,D", [("f32", 32), ("bf16", 64), ("f16", 72)])
def test_prompt_many_requests(ctx, dtype, D):
    """More requests than a block has threads, some without rows."""
    rng = np.random.default_rng(9)
    rows = rng.integers(0, 4, 900)
    rows[::50] = 0
    c = make(rng, rows, rows, dtype, 4, 2, D, lead=1, gap=2)
    got = run(ctx, c, dtype, same=True)
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, D ** -0.5,
                                      np.full(c["q"].shape, 7.0))
    assert np.abs(got - want).max() <= tolerance(dtype, s, v, 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompt_requests_do_not_meet(ctx, dtype):
    c = make(np.random.default_rng(10), [100, 30, 200], [100, 30, 200], dtype, 8, 2, 128)
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, 128 ** -0.5, c["q"])
    for x in "qkv":
        c[x][100:130] = np.nan
    got = run(ctx, c, dtype, same=True)
    rest = np.r_[0:100, 130:330]
    assert np.abs(got[rest] - want[rest]).max() <= tolerance(dtype, s, v, 200)
    assert np.isnan(got[100:130]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_prompt_large_values(ctx, dtype):
    """Scores of thousands, growing along the keys, and one of far more than the others."""
    H, K, D = 2, 1, 64
    c = make(np.random.default_rng(11), [400], [400], dtype, H, K, D)
    grow = np.linspace(0, 200, 400)
    c["k"][:, 0, 1] = ref.rounded(grow, dtype)
    c["q"][:, :, 1] = 8.0
    want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, D ** -0.5, c["q"])
    got = run(ctx, c, dtype, same=True)
    # a score's last place: 200 * 2^-24 more in the exponent, both sides
    assert np.abs(got - want).max() <= tolerance(dtype, s, v, 400)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompt_bad_starts(ctx, dtype):
    """Starts that descend or pass the buffers are cut and reported; rows of other requests
    come out right."""
    c = make(np.random.default_rng(12), [40, 30, 20], [40, 30, 20], dtype, 4, 2, 64)
    for at, value in ((3, 95), (3, 2 ** 31 - 1), (0, -5), (2, 30)):
        bad = dict(c, starts=c["starts"].copy(), ks=c["ks"].copy())
        bad["starts"][at] = bad["ks"][at] = value
        got = run(ctx, bad, dtype, same=True, bad=True)
        if at == 3:
            want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, 0.125, c["q"])
            assert np.abs(got - want).max() <= tolerance(dtype, s, v, 40)


def test_prompt_refusals(ctx):
    from chat_wgpu_b200 import CwError
    from chat_wgpu_b200.kernels.prompt import PromptAttention
    b = lambda n: ctx.storage(np.zeros(n))  # noqa: E731
    q, k, v, o = b(6 * 32), b(6 * 16), b(6 * 16), b(6 * 32)
    st = i32(ctx, [0, 2, 6])
    good = dict(q=q, k=k, v=v, starts=st, out=o, dtype="f32", n_req=2, n_rows=6, n_heads=4, n_kv=2, head_dim=8)
    PromptAttention(ctx, **good)()
    ctx.sync()
    for bad in (dict(n_req=0), dict(n_req=3), dict(n_rows=0), dict(n_rows=7), dict(n_keys=7), dict(n_keys=0),
                dict(n_heads=3), dict(n_kv=0), dict(n_heads=1), dict(head_dim=0), dict(head_dim=9),
                dict(head_dim=257), dict(window=2 ** 31), dict(softcap=-1.0), dict(softcap=float("inf")),
                dict(scale=float("nan")), dict(q_off=1), dict(k_off=1), dict(v_off=1), dict(q_stride=31),
                dict(q_stride=33), dict(k_stride=15), dict(v_stride=17), dict(q=None), dict(k=None), dict(v=None),
                dict(starts=None), dict(out=None), dict(out=q), dict(q=o), dict(k=o), dict(key_starts=b(2), n_keys=6),
                dict(key_starts=o, n_keys=6)):
        with pytest.raises(CwError) as e:
            PromptAttention(ctx, **{**good, **bad})()
        assert e.value.status == 1, bad
