"""Page plan, rotary append and tree attention on the device against the plain
64-bit forms of paged_ref.py."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def i32(ctx, a):
    return ctx.storage_u32(np.ascontiguousarray(a, np.int32).view(np.uint32))


def get(ctx, buf, n):
    return ctx.read_u32(buf, n).view(np.int32)


# ---------------------------------------------------------------- page plan
@pytest.mark.parametrize("case", [
    # (requests, cached up to, new up to, page, table slack, free share, depths, room)
    (1, 0, 1, 16, 0, 1.0, False, 0), (1, 40, 7, 16, 2, 1.0, True, 5), (8, 100, 1, 16, 1, 1.0, False, 0),
    (33, 50, 9, 1, 0, 1.0, True, 3), (513, 70, 11, 5, 1, 1.0, False, 1), (700, 300, 40, 32, 0, 0.5, False, 2),
    (40, 60, 200, 8, -3, 1.0, False, 0), (5, 30, 30, 64, 0, 0.0, False, 6), (16384, 20, 3, 16, 0, 1.0, False, 1),
    (9, 50, 60, 16, 0, 1.0, False, -37)])
def test_page_plan(ctx, case):
    from chat_wgpu_b200.kernels.pages import PagePlan
    n, cached, new, page, slack, share, deep, room = case
    rng = np.random.default_rng(n * 7 + page)
    lens = rng.integers(0, cached + 1, n).astype(np.int32)
    news = rng.integers(0, new + 1, n).astype(np.int32)
    if n > 4:
        lens[1], news[2], lens[3] = -4, -1, 0     # negative counts as 0
    c, m = np.maximum(lens, 0), np.maximum(news, 0)
    have, want = -(-c // page), -(-(c + m) // page)
    max_pages = max(1, int(want.max()) + slack)
    need = int((np.minimum(want, max_pages) - np.minimum(have, max_pages)).sum())
    n_free = int(need * share)
    ids = rng.permutation(int(have.sum()) + n_free + 1).astype(np.int32)
    table = np.full((n, max_pages), -1, np.int32)
    table[np.arange(max_pages)[None] < have[:, None]] = 0
    table[table == 0] = ids[:int((table == 0).sum())]
    free = ids[len(ids) - n_free:]
    max_tokens = max(1, int(m.sum()) + room)
    depths = rng.integers(0, 9, max_tokens).astype(np.int32) if deep else None
    t = i32(ctx, table)
    out = {k: i32(ctx, np.full(s, -77)) for k, s in dict(
        starts=n + 1, positions=max_tokens, slots=max_tokens, owners=max_tokens, used=1).items()}
    call = PagePlan(ctx, lens=i32(ctx, lens), news=i32(ctx, news), free_pages=i32(ctx, free) if n_free else None,
                    table=t, depths=i32(ctx, depths) if deep else None, n_req=n, page_size=page,
                    max_pages=max_pages, n_free=n_free, max_tokens=max_tokens, **out)
    want_ = ref.plan(lens, news, free, table, page, max_tokens, depths)
    for _ in range(2):  # planning the same step again gives the same pages
        call()
        assert int(get(ctx, out["used"], 1)[0]) == want_["used"]
        assert np.array_equal(get(ctx, out["starts"], n + 1), want_["starts"])
        assert np.array_equal(get(ctx, t, table.size).reshape(table.shape), want_["table"])
        for k in ("positions", "slots", "owners"):
            assert np.array_equal(get(ctx, out[k], max_tokens), want_[k]), k


def test_page_plan_refusals(ctx):
    from chat_wgpu_b200 import CwError
    from chat_wgpu_b200.kernels.pages import PagePlan
    b = i32(ctx, np.zeros(64))
    good = dict(lens=b, news=b, free_pages=b, table=b, starts=b, positions=b, slots=b, owners=b, used=b,
                n_req=2, page_size=16, max_pages=4, n_free=4, max_tokens=8)
    PagePlan(ctx, **good)()
    for bad in (dict(n_req=0), dict(n_req=16385), dict(page_size=0), dict(max_pages=0), dict(max_pages=33),
                dict(n_free=65), dict(max_tokens=65), dict(n_req=64), dict(lens=None), dict(used=None)):
        with pytest.raises(CwError) as e:
            PagePlan(ctx, **{**good, **bad})()
        assert e.value.status == 1, bad


# ---------------------------------------------------------------- rotary append
ROPE = [  # dtype, T, H, K, D, rot, layout, scaling, page, fused (q, k, v in one row)
    ("f32", 1, 4, 2, 16, 16, "half", dict(), 16, False),
    ("f32", 37, 16, 8, 128, 128, "half", dict(), 16, True),
    ("f32", 70, 3, 3, 33, 22, "half", dict(kind="linear", factor=4.0), 5, False),
    ("f32", 5, 2, 1, 10, 6, "interleaved", dict(), 1, True),
    ("f16", 67, 8, 4, 256, 64, "interleaved", dict(kind="yarn", factor=4.0, low=1.0, high=32.0, trained=32768), 16, False),
    ("f16", 300, 24, 8, 80, 60, "half", dict(kind="yarn", factor=8.0, low=1.0, high=32.0, trained=4096, amplitude=1.25), 8, True),
    ("bf16", 129, 32, 8, 128, 128, "half", dict(kind="banded", factor=8.0, low=1.0, high=4.0, trained=8192), 32, True),
    ("bf16", 2, 7, 7, 96, 72, "interleaved", dict(), 64, False),
    ("bf16", 2000, 32, 8, 128, 64, "interleaved", dict(), 64, True),
    ("f16", 9, 1, 1, 7, 2, "half", dict(), 3, False),
]


@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(map(str, c[:7])))
def test_rope_append(ctx, case):
    from chat_wgpu_b200.kernels.rope import RopeAppend, rope_plan
    dtype, T, H, K, D, rot, layout, scaling, page, fused = case
    rng = np.random.default_rng(T + D)
    es = 16 // ref.SIZE[dtype]
    wq, wk = H * D, K * D
    if fused:
        rows = ref.rounded(rng.normal(0, 1, (T, wq + 2 * wk)), dtype)
        src = ref.upload(ctx, rows, dtype)
        q, k, v = rows[:, :wq], rows[:, wq:wq + wk], rows[:, wq + wk:]
        where = dict(q=src, k=src, v=src, k_off=wq, v_off=wq + wk, q_stride=wq + 2 * wk,
                     k_stride=wq + 2 * wk, v_stride=wq + 2 * wk)
    else:
        q, k, v = (ref.rounded(rng.normal(0, 1, (T, w)), dtype) for w in (wq, wk, wk))
        where = dict(q=ref.upload(ctx, q, dtype), k=ref.upload(ctx, k, dtype), v=ref.upload(ctx, v, dtype))
    n_pages = -(-T // page) + 2
    pos = rng.integers(0, 200000, T).astype(np.int32)
    pos[0] = 0
    slots = rng.permutation(n_pages * page)[:T].astype(np.int32)
    if T > 3:
        slots[1] = -1
    shape = (n_pages, K, page, D)
    old = [ref.rounded(rng.normal(0, 1, shape), dtype) for _ in range(2)]
    kc, vc = (ref.upload(ctx, x, dtype) for x in old)
    out = ref.upload(ctx, np.zeros((T, wq)), dtype)
    plan = rope_plan(ctx, rot, 1e4, **scaling)
    RopeAppend(ctx, plan=plan, positions=i32(ctx, pos), dtype=dtype, layout=layout, n_tokens=T, n_heads=H,
               n_kv=K, head_dim=D, q_out=out, slots=i32(ctx, slots), k_cache=kc, v_cache=vc, page_size=page,
               n_pages=n_pages, **where)()
    f, amp = ref.rates(rot, 1e4, **scaling)
    # a rotated value: the angle is exact to 2^-24 of half a turn (2 pi 2^-25), sine and
    # cosine to 2 units, the two products and their sum to 1 unit each, on |x0| + |x1|;
    # then one rounding to the type.  The reference's own angle in f64 is off by
    # 200000 * 2^-53 * a few, below 2^-33.
    most = 2 * amp * max(np.abs(q).max(), np.abs(k).max())
    tol = most * (6 * 2.0 ** -24 + 2 * np.pi * 2.0 ** -25) + (ref.UNIT[dtype] * most if dtype != "f32" else 0)
    got = ref.read(ctx, out, dtype, (T, H, D))
    assert np.abs(got - ref.rotate(q.reshape(T, H, D), pos, f, amp, layout)).max() <= tol
    kr = ref.rotate(k.reshape(T, K, D), pos, f, amp, layout)
    want_k, want_v = old[0].copy(), old[1].copy()
    for t in range(T):
        if slots[t] >= 0:
            want_k[slots[t] // page, :, slots[t] % page] = kr[t]
            want_v[slots[t] // page, :, slots[t] % page] = v.reshape(T, K, D)[t]
    assert np.array_equal(ref.read(ctx, vc, dtype, shape), want_v)
    gk = ref.read(ctx, kc, dtype, shape)
    assert np.abs(gk - want_k).max() <= tol
    touched = np.zeros((n_pages, page), bool)
    live = slots[slots >= 0]
    touched[live // page, live % page] = True
    keep = ~touched[:, None, :, None] & np.ones(shape, bool)
    assert np.array_equal(gk[keep], old[0][keep])


def test_rope_parts_and_place(ctx):
    """q alone in place, k and v alone, negative positions, values that are not finite."""
    from chat_wgpu_b200.kernels.rope import RopeAppend, rope_plan
    T, H, K, D, page = 6, 4, 2, 16, 4
    rng = np.random.default_rng(3)
    q, k, v = (rng.normal(0, 1, (T, n * D)).astype(np.float32) for n in (H, K, K))
    q[2, 12] = np.inf      # past the rotated 8 elements: passes through
    v[1, 3] = np.nan
    pos = np.array([0, 5, -3, 1, 2, 7], np.int32)
    plan = rope_plan(ctx, 8, 1e4)
    qb, pb = ctx.storage(q), i32(ctx, pos)
    RopeAppend(ctx, plan=plan, positions=pb, dtype="f32", n_tokens=T, n_heads=H, head_dim=D, q=qb, q_out=qb)()
    f, amp = ref.rates(8, 1e4)
    want = ref.rotate(q.reshape(T, H, D).astype(np.float64), pos, f, amp, "half").reshape(T, -1)
    got = ctx.read(qb, q.size).reshape(q.shape)
    fine = np.isfinite(want)
    assert got[2, 12] == np.inf and np.abs(got[fine] - want[fine]).max() < 1e-5
    kc, vc = ctx.storage(np.zeros(3 * K * page * D)), ctx.storage(np.zeros(3 * K * page * D))
    RopeAppend(ctx, plan=plan, positions=pb, dtype="f32", n_tokens=T, n_kv=K, head_dim=D, k=ctx.storage(k),
               v=ctx.storage(v), slots=i32(ctx, np.arange(T) + 3), k_cache=kc, v_cache=vc, page_size=page,
               n_pages=3)()
    got = ctx.read(vc, 3 * K * page * D).reshape(3, K, page, D)
    for t in range(T):
        assert np.array_equal(got[(t + 3) // page, :, (t + 3) % page].ravel(), v[t], equal_nan=True)


def test_rope_refusals(ctx):
    from chat_wgpu_b200 import CwError
    from chat_wgpu_b200.kernels.rope import RopeAppend, rope_plan
    z, s = ctx.storage(np.zeros(4096)), i32(ctx, np.zeros(64))
    plan = rope_plan(ctx, 16, 1e4)
    good = dict(plan=plan, positions=s, dtype="f32", n_tokens=4, n_heads=4, n_kv=2, head_dim=16, q=z, q_out=z,
                k=z, v=z, slots=s, k_cache=z, v_cache=z, page_size=16, n_pages=2)
    for bad in (dict(n_tokens=0), dict(head_dim=8), dict(plan=z), dict(n_heads=0, n_kv=0), dict(page_size=0),
                dict(n_pages=1000), dict(q_stride=63), dict(k_stride=31), dict(q_off=5), dict(n_tokens=65),
                dict(k=None), dict(head_dim=2048)):
        with pytest.raises(CwError) as e:
            RopeAppend(ctx, **{**good, **bad})()
        assert e.value.status == 1, bad
    with pytest.raises(ValueError):
        RopeAppend(ctx, **{**good, "dtype": "f64"})
    for bad in (dict(rot_dim=0), dict(rot_dim=7), dict(theta=0.5), dict(theta=float("inf")),
                dict(kind="linear", factor=0.0), dict(kind="banded", factor=2.0, low=4.0, high=1.0, trained=10),
                dict(kind="yarn", factor=2.0, trained=0)):
        with pytest.raises(CwError) as e:
            rope_plan(ctx, **{**dict(rot_dim=16, theta=1e4), **bad})
        assert e.value.status == 1, bad
    # a slot outside the cache is skipped and reported, and the context stays usable
    c = ctx.storage(np.zeros(2 * 2 * 16 * 16))
    RopeAppend(ctx, **{**good, "slots": i32(ctx, [0, 32, 1, 2]), "k_cache": c, "v_cache": c})()
    with pytest.raises(CwError) as e:
        ctx.sync()
    assert e.value.status == 1
    ctx.sync()


# ---------------------------------------------------------------- tree attention
def tree_case(rng, lens, nodes, dtype, H, K, D, page, empty=False, poison=True):
    """Random trees over a paged cache whose unused places hold NaN."""
    n = len(lens)
    lens, nodes = np.array(lens, np.int32), np.array(nodes, np.int32)
    starts = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    T, N = int(starts[-1]), max(1, int(nodes.max()))
    used = -(-(lens + nodes) // page)
    max_pages, n_pages = max(1, int(used.max())) + 1, int(used.sum()) + 3
    ids = rng.permutation(n_pages)
    table = np.full((n, max_pages), -1, np.int32)
    table[np.arange(max_pages)[None] < used[:, None]] = ids[:int(used.sum())]
    shape = (n_pages, K, page, D)
    kc, vc = (ref.rounded(rng.normal(0, 1, shape), dtype) for _ in range(2))
    live = np.zeros((n_pages, page), bool)
    see, pos = [], np.zeros(max(T, 1), np.int32)
    for r in range(n):
        at = np.arange(lens[r] + nodes[r])
        live[table[r, at // page], at % page] = True
        m = int(nodes[r])
        s, depth = np.zeros((m, m), bool), np.zeros(m, int)
        for i in range(m):
            if i and rng.random() < 0.9:
                parent = int(rng.integers(0, i))
                s[i], depth[i] = s[parent], depth[parent] + 1
            s[i, i] = True
        if empty and m:
            s[rng.random(m) < 0.3] = False
        see.append(s)
        pos[starts[r]:starts[r] + m] = lens[r] + depth
        if poison and m > 2:  # a node that only itself sees holds values that are not finite
            j = m - 1
            s[:j, j] = False
            page_j, off_j = table[r, (lens[r] + j) // page], (lens[r] + j) % page
            s[j] = False                       # and now nobody does
            kc[page_j, :, off_j], vc[page_j, :, off_j] = np.nan, np.inf
    dead = np.broadcast_to(~live[:, None, :, None], shape)
    kc[dead], vc[dead] = np.nan, np.nan
    words = -(-N // 32)
    mask = np.zeros((max(T, 1), words * 32), np.uint8)
    for r in range(n):
        mask[starts[r]:starts[r + 1], :nodes[r]] = see[r]
    mask = np.packbits(mask, axis=1, bitorder="little").view(np.uint32)
    q = ref.rounded(rng.normal(0, 2, (max(T, 1), H, D)), dtype)
    return dict(lens=lens, starts=starts, T=T, N=N, table=table, kc=kc, vc=vc, see=see, pos=pos, mask=mask,
                q=q, max_pages=max_pages, n_pages=n_pages)


def tree_run(ctx, c, dtype, H, K, D, page, window=0, softcap=0.0, scale=0.0, mask=True, pad=0, off=0):
    from chat_wgpu_b200.kernels.tree import TreeAttention
    T = max(c["T"], 1)
    rows = np.full((T, H * D + pad), np.nan)
    rows[:, off:off + H * D] = c["q"].reshape(T, -1)
    out = ref.upload(ctx, np.full((T, H, D), 7.0), dtype)
    TreeAttention(ctx, q=ref.upload(ctx, rows, dtype), k_cache=ref.upload(ctx, c["kc"], dtype),
                  v_cache=ref.upload(ctx, c["vc"], dtype), table=i32(ctx, c["table"]), lens=i32(ctx, c["lens"]),
                  starts=i32(ctx, c["starts"]), mask=ctx.storage_u32(c["mask"]) if mask else None,
                  positions=i32(ctx, c["pos"]), out=out, dtype=dtype, n_req=len(c["lens"]), n_rows=T,
                  max_nodes=c["N"], n_heads=H, n_kv=K, head_dim=D, page_size=page, n_pages=c["n_pages"],
                  max_pages=c["max_pages"], window=window, softcap=softcap, scale=scale,
                  q_off=off, q_stride=H * D + pad)()
    return ref.read(ctx, out, dtype, (T, H, D))


def tree_tolerance(dtype, big_s, big_v):
    """A score's products carry 2^-21 each (two split operands and the dropped term) and
    its f32 sum 2^-24 per addition pair, so a score is off by at most 2^-19 of the sum of
    its terms' magnitudes; weights move by twice that, the exponential, the running
    rescales and the join by 2^-18; a 16-bit type rounds each weight once (u) and the
    result once (u).  All on values of at most big_v."""
    u = 0.0 if dtype == "f32" else ref.UNIT[dtype]
    return big_v * (2 * 2.0 ** -19 * big_s + 2.0 ** -18 + 2 * u)


TREE = [  # dtype, heads, kv, dim, page, lens, nodes, options
    ("f32", 4, 2, 16, 16, [0], [1], {}),
    ("f32", 16, 8, 128, 16, [1037], [1], {}),
    ("f32", 4, 2, 64, 5, [0, 1, 63, 64, 65, 127, 200], [1, 3, 1, 5, 0, 33, 9], {}),
    ("f32", 16, 8, 128, 16, [300, 64, 700], [24, 17, 8], {}),
    ("f32", 8, 4, 256, 64, [130, 5], [13, 40], dict(window=50, softcap=20.0)),
    ("f32", 7, 7, 33, 3, [40, 0], [6, 4], {}),
    ("f32", 8, 1, 80, 7, [90], [70], dict(window=3)),
    ("f32", 2, 1, 128, 16, [5000], [2], {}),
    ("f32", 4, 4, 32, 16, [10, 100], [100, 65], dict(empty=True)),
    ("f16", 4, 2, 64, 16, [0, 1, 63, 64, 65, 127, 200], [1, 3, 1, 5, 0, 33, 9], {}),
    ("f16", 8, 4, 256, 64, [500, 70, 0], [13, 9, 5], dict(window=200, softcap=50.0)),
    ("f16", 8, 4, 256, 16, [1000], [20], {}),
    ("f16", 16, 8, 64, 32, [900, 31, 33], [1, 1, 1], {}),
    ("f16", 12, 4, 96, 8, [77, 400], [31, 64], dict(empty=True)),
    ("f16", 4, 2, 36, 16, [100], [9], {}),
    ("f16", 3, 1, 128, 5, [61, 400], [9, 2], {}),
    ("bf16", 32, 8, 128, 16, [700, 130, 64, 1], [16, 7, 1, 2], {}),
    ("bf16", 32, 8, 128, 64, [3000, 100], [64, 33], {}),
    ("bf16", 32, 8, 128, 128, [200], [100], dict(softcap=30.0, window=90)),
    ("bf16", 8, 8, 48, 16, [250, 10], [5, 4], dict(empty=True)),
    ("bf16", 16, 2, 64, 256, [1000], [200], {}),
    ("bf16", 24, 8, 80, 32, [333], [12], {}),
    ("bf16", 1, 1, 8, 8, [9, 0, 2], [1, 0, 3], {}),
    ("bf16", 8, 4, 64, 192, [1000, 100], [4, 30], {}),
    ("f16", 16, 2, 128, 320, [1500], [12], {}),
    # several tiles to a block's run, for each way a tile's keys are dealt to the lanes
    ("bf16", 8, 8, 128, 64, [6000], [1], {}),
    ("bf16", 32, 8, 128, 16, [4000, 900], [8, 3], {}),
    ("bf16", 32, 8, 128, 64, [5000], [9], {}),
    ("f16", 32, 8, 64, 32, [4500, 40], [16, 12], dict(softcap=10.0)),
    ("f16", 32, 8, 64, 8, [4500], [33], dict(window=1000)),
    ("f16", 8, 4, 256, 64, [6000], [40], {}),
    ("bf16", 32, 8, 128, 16, [3000, 70], [25, 31], {}),
    ("f16", 16, 4, 48, 32, [3500], [30], dict(window=700, softcap=15.0)),
    ("bf16", 16, 8, 200, 8, [2000], [5], {}),
    ("f16", 8, 4, 256, 16, [900, 3000], [30, 64], dict(empty=True)),
    ("f32", 16, 8, 128, 16, [3000, 700], [9, 30], {}),
]


@pytest.mark.parametrize("case", TREE, ids=lambda c: f"{c[0]}-{c[1]}x{c[2]}x{c[3]}-p{c[4]}-{max(c[5])}x{max(c[6])}")
def test_tree_attention(ctx, case):
    dtype, H, K, D, page, lens, nodes, opt = case
    opt = dict(opt)
    rng = np.random.default_rng(sum(lens) + D)
    c = tree_case(rng, lens, nodes, dtype, H, K, D, page, empty=opt.pop("empty", False))
    got = tree_run(ctx, c, dtype, H, K, D, page, pad=24, off=8, **opt)
    want, s, v = ref.attention(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], page, c["see"],
                               c["pos"], opt.get("window", 0), opt.get("softcap", 0.0), D ** -0.5)
    assert np.isfinite(got).all()
    assert np.abs(got - want).max() <= tree_tolerance(dtype, s, v)
    ctx.sync()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_tree_chain_and_scale(ctx, dtype):
    """No mask: node i sees nodes 0..i.  A given scale.  Bits of two runs are the same."""
    H, K, D, page = 8, 2, 64, 16
    c = tree_case(np.random.default_rng(5), [100, 0], [37, 70], dtype, H, K, D, page, poison=False)
    see = [np.tril(np.ones((m, m), bool)) for m in (37, 70)]
    got = tree_run(ctx, c, dtype, H, K, D, page, scale=0.3, mask=False)
    want, s, v = ref.attention(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], page, see, c["pos"],
                               0, 0.0, 0.3)
    assert np.abs(got - want).max() <= tree_tolerance(dtype, s, v)
    again = tree_run(ctx, c, dtype, H, K, D, page, scale=0.3, mask=False)
    assert np.array_equal(got, again)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tree_visible_not_finite(ctx, dtype):
    """A value that is not finite reaches the rows that see it and no others."""
    H, K, D, page = 4, 2, 64, 16
    c = tree_case(np.random.default_rng(6), [70], [5], dtype, H, K, D, page, poison=False)
    c["see"] = [np.tril(np.ones((5, 5), bool))]
    for at in (72, 74):  # nodes 2 and 4
        c["vc"][c["table"][0, at // page], 1, at % page, 3] = np.inf if at == 72 else np.nan
    got = tree_run(ctx, c, dtype, H, K, D, page, mask=False)
    assert np.isfinite(got[:2]).all() and np.isfinite(got[:, :2]).all()
    assert (got[2:4, 2:, 3] == np.inf).all() and np.isnan(got[4, 2:, 3]).all()
    rest = np.ones(D, bool)
    rest[3] = False
    assert np.isfinite(got[:, :, rest]).all()


@pytest.mark.parametrize("dtype,D,page", [("f32", 32, 8), ("bf16", 64, 8), ("f16", 72, 5)])
def test_tree_many_requests(ctx, dtype, D, page):
    """More requests than a block has threads, some without tokens or without nodes."""
    H, K = 2, 1
    rng = np.random.default_rng(9)
    lens, nodes = rng.integers(0, 40, 700), rng.integers(0, 3, 700)
    lens[::50] = 0
    c = tree_case(rng, lens, nodes, dtype, H, K, D, page)
    got = tree_run(ctx, c, dtype, H, K, D, page)
    want, s, v = ref.attention(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], page, c["see"],
                               c["pos"], 0, 0.0, D ** -0.5)
    assert np.abs(got - want).max() <= tree_tolerance(dtype, s, v)
    ctx.sync()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tree_requests_do_not_meet(ctx, dtype):
    """Queries of one request that are not finite leave the others' rows alone."""
    H, K, D, page = 8, 2, 128, 16
    c = tree_case(np.random.default_rng(10), [200, 30, 300], [3, 16, 7], dtype, H, K, D, page)
    want, s, v = ref.attention(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], page, c["see"],
                               c["pos"], 0, 0.0, D ** -0.5)
    c["q"][3:19] = np.nan
    got = tree_run(ctx, c, dtype, H, K, D, page)
    rest = np.r_[0:3, 19:26]
    assert np.abs(got[rest] - want[rest]).max() <= tree_tolerance(dtype, s, v)


@pytest.mark.parametrize("dtype,pages", [("bf16", 70000), ("f32", 36000)])
def test_far_pages(ctx, dtype, pages):
    """Pages whose elements lie past 32 bits (bf16: 4.6e9 elements, f32: 2.4e9) hold and
    give back the same as pages at the start."""
    torch = pytest.importorskip("torch")
    from chat_wgpu_b200 import GpuContext
    from chat_wgpu_b200.kernels import rope, tree
    H, K, D, page, T, n = 8, 8, 128, 64, 150, 3
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    q, k, v = rnd(T, H * D), rnd(T, K * D), rnd(T, K * D)
    kc, vc = (torch.empty(pages, K, page, D, dtype=dt, device="cuda") for _ in range(2))
    c = GpuContext(0, stream=torch.cuda.current_stream().cuda_stream)
    plan = rope.rope_plan(c, D, 1e4)
    kw, vw, pos, outs = c.wrap(kc), c.wrap(vc), c.wrap(i(range(T))), []
    for first in (0, pages - n):
        slots = c.wrap(i([first * page + t for t in range(T)]))
        rot = torch.empty_like(q)
        rope.RopeAppend(c, plan=plan, positions=pos, dtype=dtype, n_tokens=T, n_heads=H, n_kv=K, head_dim=D,
                        q=c.wrap(q), q_out=c.wrap(rot), k=c.wrap(k), v=c.wrap(v), slots=slots, k_cache=kw,
                        v_cache=vw, page_size=page, n_pages=pages)()
        out = torch.empty(5, H * D, dtype=dt, device="cuda")
        tree.TreeAttention(c, q=c.wrap(rot[:5]), k_cache=kw, v_cache=vw, table=c.wrap(i([[first, first + 1, first + 2]])),
                           lens=c.wrap(i([T - 5])), starts=c.wrap(i([0, 5])), out=c.wrap(out), dtype=dtype, n_req=1,
                           n_rows=5, max_nodes=5, n_heads=H, n_kv=K, head_dim=D, page_size=page, n_pages=pages,
                           max_pages=n)()
        c.sync()
        assert torch.equal(vc[first + 1].transpose(0, 1).reshape(page, -1), v[page:2 * page])
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and bool(outs[0].isfinite().all())
    c.close()
    del kc, vc
    torch.cuda.empty_cache()


def test_tree_no_rows(ctx):
    """A step in which no request has nodes writes nothing."""
    c = tree_case(np.random.default_rng(11), [20, 3], [0, 0], "bf16", 4, 2, 64, 16)
    assert (tree_run(ctx, c, "bf16", 4, 2, 64, 16) == 7.0).all()
    ctx.sync()


def test_tree_refusals(ctx):
    from chat_wgpu_b200 import CwError
    from chat_wgpu_b200.kernels.tree import TreeAttention
    z, s = ctx.storage(np.zeros(8192)), i32(ctx, np.zeros(64))
    good = dict(q=z, k_cache=z, v_cache=z, table=s, lens=s, starts=i32(ctx, [0, 1, 2]), mask=s, positions=s, out=z,
                dtype="f32", n_req=2, n_rows=2, max_nodes=2, n_heads=4, n_kv=2, head_dim=16, page_size=16,
                n_pages=2, max_pages=2)
    TreeAttention(ctx, **good)()
    ctx.sync()
    for bad in (dict(n_heads=5), dict(n_kv=0), dict(head_dim=0), dict(head_dim=257), dict(max_nodes=0),
                dict(max_nodes=1025), dict(n_req=0), dict(n_rows=0), dict(page_size=0), dict(n_pages=100),
                dict(max_pages=33), dict(q_stride=63), dict(q_off=8100), dict(n_rows=4000), dict(scale=-1.0),
                dict(softcap=-1.0), dict(softcap=float("nan")), dict(out=None), dict(window=4, positions=None)):
        with pytest.raises(CwError) as e:
            TreeAttention(ctx, **{**good, **bad})()
        assert e.value.status == 1, bad
    # device data out of range: skipped, reported once, the context stays usable
    for bad in (dict(table=i32(ctx, np.full(4, 9))), dict(starts=i32(ctx, [0, 5, 2])), dict(lens=i32(ctx, [40, 0])),
                dict(lens=i32(ctx, [-1, 0]))):
        TreeAttention(ctx, **{**good, **bad})()
        with pytest.raises(CwError) as e:
            ctx.sync()
        assert e.value.status == 1
        ctx.sync()


# ---------------------------------------------------------------- another library's tensors
def test_wrapped_tensors_and_stream(ctx):
    """Tensors of torch as buffers, on torch's stream, without copies."""
    torch = pytest.importorskip("torch")
    from chat_wgpu_b200 import CwError, GpuContext
    from chat_wgpu_b200.kernels import attention
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c = GpuContext(0, stream=side.cuda_stream)
        a, b = torch.arange(1000, device="cuda", dtype=torch.float32), torch.full((1000,), 2.0, device="cuda")
        wa, wb = c.wrap(a), c.wrap(b)
        assert wa.nbytes == 4000 and wa.device_ptr == a.data_ptr()
        out = torch.zeros(1000, device="cuda")
        wo = c.wrap(out)
        for _ in range(3):   # torch and the library in turn on one stream
            a.add_(1.0)
            c.copy(attention.add(c, wa, wb, 1000), 0, wo, 0, 1000)
            b.copy_(out)
            c.reset_frame()
    side.synchronize()
    assert torch.equal(b.cpu(), 3 * torch.arange(1000.0) + 2 + 1 + 2 + 3)
    strided = torch.zeros(4, 64, device="cuda")[:, 16:32]
    assert c.wrap(strided).nbytes == (3 * 64 + 16) * 4
    with pytest.raises(CwError):
        c.wrap(a[1:])            # 4 bytes past a 16-byte boundary
    with pytest.raises(CwError):
        c.wrap(torch.zeros(8))   # host memory
    wa.release()
    assert float(a[5]) == 8.0    # the memory is still the tensor's
    c.close()
    assert float(a[6]) == 9.0
