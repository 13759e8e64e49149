"""Head norms, rotation and append in one pass on the device against the 64-bit form."""
import numpy as np
import pytest

import paged_ref as ref
import prompt_ref

pytestmark = pytest.mark.gpu


def i32(ctx, a):
    return ctx.storage_u32(np.ascontiguousarray(a, np.int32).view(np.uint32))


CASES = [  # dtype, T, H, K, D, rot, layout, shift, page (0: no cache), k_out, fused, norms
    ("f32", 1, 16, 8, 128, 128, "half", False, 16, False, True, "qk"),
    ("f32", 1, 1, 1, 2, 2, "half", False, 0, True, False, "qk"),
    ("f32", 37, 16, 8, 128, 128, "half", False, 16, True, True, "qk"),
    ("f32", 70, 3, 3, 33, 22, "half", True, 5, True, False, "qk"),
    ("f32", 5, 2, 1, 10, 6, "interleaved", False, 1, False, True, "k"),
    ("f32", 9, 2, 2, 1024, 512, "half", False, 16, True, False, "qk"),
    ("f32", 3, 2, 1, 1023, 2, "interleaved", False, 4, True, True, "qk"),
    ("f16", 67, 8, 4, 256, 64, "interleaved", True, 16, True, False, "qk"),
    ("f16", 300, 24, 8, 80, 60, "half", False, 8, False, True, "q"),
    ("f16", 9, 1, 1, 7, 2, "half", False, 3, True, False, "qk"),
    ("f16", 11, 2, 2, 1000, 8, "half", False, 16, True, False, "qk"),
    ("bf16", 129, 32, 8, 128, 128, "half", False, 32, False, True, "qk"),
    ("bf16", 2, 7, 7, 96, 72, "interleaved", False, 64, True, False, "qk"),
    ("bf16", 2000, 32, 8, 128, 64, "interleaved", False, 64, False, True, "qk"),
    ("bf16", 31, 4, 0, 64, 64, "half", False, 0, False, False, "qk"),
    ("bf16", 31, 0, 4, 64, 32, "half", False, 16, False, False, "qk"),
    ("bf16", 6, 8, 4, 64, 64, "half", False, 8, True, False, ""),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:7])))
def test_norm_rope(ctx, case):
    from chat_wgpu_b200.kernels.rope import NormRope, rope_plan
    dtype, T, H, K, D, rot, layout, shift, page, k_out, fused, norms = case
    rng = np.random.default_rng(T + D)
    wq, wk, eps = H * D, K * D, 1e-6
    scale = np.exp2(rng.integers(-3, 4, (T, 1)))  # rows of different sizes
    rows = ref.rounded(rng.normal(0, 1, (T, wq + 2 * wk)) * scale, dtype)
    q, k, v = rows[:, :wq], rows[:, wq:wq + wk], rows[:, wq + wk:]
    if fused:
        src = ref.upload(ctx, rows, dtype)
        where = dict(q=src, k=src, v=src, k_off=wq, v_off=wq + wk, q_stride=wq + 2 * wk,
                     k_stride=wq + 2 * wk, v_stride=wq + 2 * wk)
    else:
        where = {n: ref.upload(ctx, x, dtype) for n, x in (("q", q), ("k", k), ("v", v)) if x.size}
    pos = rng.integers(0, 200000, T).astype(np.int32)
    pos[0] = 0
    w = {n: rng.normal(0 if shift else 1, 0.3, D).astype(np.float32) if n in norms else None for n in "qk"}
    n_pages = -(-T // max(page, 1)) + 2
    shape = (n_pages, K, page, D)
    old = [ref.rounded(rng.normal(0, 1, shape), dtype) for _ in range(2)]
    slots = rng.permutation(n_pages * max(page, 1))[:T].astype(np.int32)
    if T > 3:
        slots[1] = -1
    more = {}
    if page and K:
        more = dict(slots=i32(ctx, slots), k_cache=ref.upload(ctx, old[0], dtype),
                    v_cache=ref.upload(ctx, old[1], dtype), page_size=page, n_pages=n_pages)
    out = {n: ref.upload(ctx, np.full((T, x), 7.0), dtype) for n, x in (("q_out", wq), ("k_out", wk))
           if x and (n == "q_out" or k_out)}
    plan = rope_plan(ctx, rot, 1e4)
    NormRope(ctx, plan=plan, positions=i32(ctx, pos), dtype=dtype, n_tokens=T, head_dim=D, eps=eps,
             unit_shift=shift, layout=layout, n_heads=H, n_kv=K, **where, **more, **out,
             **{n + "_norm": ctx.storage(x) for n, x in w.items() if x is not None})()
    ctx.sync()
    f, amp = ref.rates(rot, 1e4)
    # the norm: a sum of D squares in at most 32 + 5 roundings along any path, half of that
    # in the root, root, quotient and two products 1 unit each: 24 units of 2^-24.  The
    # rotation: angle 2^-24 of half a turn, sine and cosine 2 units (2^-21 in 16-bit types),
    # products and sum 1 unit each, on |x0| + |x1|; then one rounding to the type.
    sines = 2.0 ** -21 if dtype != "f32" else 2 * 2.0 ** -24

    def check(got, x, heads, weight):
        want = prompt_ref.norm_rotate(x.reshape(T, heads, D), weight, shift, eps, pos, f, amp, layout)
        plain = prompt_ref.norm_rotate(x.reshape(T, heads, D), weight, shift, eps, pos * 0, f, amp, layout)
        most = 2 * np.abs(plain).max(-1, keepdims=True)
        tol = most * (24 * 2.0 ** -24 + sines + 3 * 2.0 ** -24 + 2 * np.pi * 2.0 ** -25)
        if dtype != "f32":
            tol = tol + ref.UNIT[dtype] * np.abs(want) + 2.0 ** -25 * (dtype == "f16")
        assert (np.abs(got - want) <= tol).all()
        return want

    if H:
        check(ref.read(ctx, out["q_out"], dtype, (T, H, D)), q, H, w["q"])
    if K:
        if k_out:
            check(ref.read(ctx, out["k_out"], dtype, (T, K, D)), k, K, w["k"])
        if page:
            kc, vc = (ref.read(ctx, more[n], dtype, shape) for n in ("k_cache", "v_cache"))
            at = np.flatnonzero(slots >= 0)
            got = np.zeros((T, K, D))
            got[at] = kc[slots[at] // page, :, slots[at] % page]
            if k_out:
                assert np.array_equal(got[at], ref.read(ctx, out["k_out"], dtype, (T, K, D))[at])
            else:
                want = prompt_ref.norm_rotate(k.reshape(T, K, D), w["k"], shift, eps, pos, f, amp, layout)
                got[slots < 0] = want[slots < 0]
                check(got, k, K, w["k"])
            want_v = old[1].copy()
            want_v[slots[at] // page, :, slots[at] % page] = v.reshape(T, K, D)[at]
            assert np.array_equal(vc, want_v)
            kept = np.ones((n_pages, page), bool)
            kept[slots[at] // page, slots[at] % page] = False
            kept = np.broadcast_to(kept[:, None, :, None], shape)
            assert np.array_equal(kc[kept], old[0][kept])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_rope_in_place_and_again(ctx, dtype):
    """Contiguous rows in place give the bits of rows written elsewhere; a zero row stays zero."""
    from chat_wgpu_b200.kernels.rope import NormRope, rope_plan
    T, H, K, D = 45, 6, 2, 64
    rng = np.random.default_rng(3)
    q, k = (ref.rounded(rng.normal(0, 2, (T, n * D)), dtype) for n in (H, K))
    q[7] = 0
    pos, plan = i32(ctx, rng.integers(0, 5000, T)), rope_plan(ctx, D, 1e6)
    w = ctx.storage(rng.normal(1, 0.2, D))

    def run(qo, ko, qi, ki):
        NormRope(ctx, plan=plan, positions=pos, dtype=dtype, n_tokens=T, head_dim=D, eps=1e-5, n_heads=H,
                 n_kv=K, q=qi, q_norm=w, q_out=qo, k=ki, k_norm=w, k_out=ko)()
        return ref.read(ctx, qo, dtype, (T, H * D)), ref.read(ctx, ko, dtype, (T, K * D))

    new = lambda n: ref.upload(ctx, np.zeros((T, n * D)), dtype)  # noqa: E731
    a = run(new(H), new(K), ref.upload(ctx, q, dtype), ref.upload(ctx, k, dtype))
    qi, ki = ref.upload(ctx, q, dtype), ref.upload(ctx, k, dtype)
    b = run(qi, ki, qi, ki)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    assert not a[0][7].any()


def test_norm_rope_not_finite(ctx):
    """Heads that are not finite, or too large for f32 squares, leave other heads alone."""
    from chat_wgpu_b200.kernels.rope import NormRope, rope_plan
    T, H, D = 3, 4, 64
    q = np.random.default_rng(4).normal(0, 1, (T, H, D)).astype(np.float32)
    want = q.copy()
    q[1, 1, 5], q[1, 2, 6], q[2, 0, 0] = np.nan, np.inf, 1e30
    out = ctx.storage(np.zeros(q.size))
    NormRope(ctx, plan=rope_plan(ctx, D, 1e4), positions=i32(ctx, [0, 0, 0]), dtype="f32", n_tokens=T,
             head_dim=D, eps=0.0, n_heads=H, q=ctx.storage(q), q_norm=ctx.storage(np.ones(D)), q_out=out)()
    got = ctx.read(out, q.size).reshape(q.shape)
    want /= np.sqrt((want.astype(np.float64) ** 2).mean(-1, keepdims=True))
    rest = np.ones((T, H), bool)
    rest[1, 1] = rest[1, 2] = rest[2, 0] = False
    assert np.isnan(got[1, 1]).all()
    assert np.abs(got[rest] - want[rest]).max() <= 24 * 2.0 ** -24 * np.abs(want[rest]).max()


def test_norm_rope_refusals(ctx):
    from chat_wgpu_b200 import CwError
    from chat_wgpu_b200.kernels.rope import NormRope, rope_plan
    b = lambda n: ctx.storage(np.zeros(n))  # noqa: E731
    T, H, K, D = 4, 2, 1, 8
    plan, pos, slots = rope_plan(ctx, D, 1e4), i32(ctx, np.zeros(T)), i32(ctx, np.arange(T))
    q, k, v, qo, ko = b(T * H * D), b(T * K * D), b(T * K * D), b(T * H * D), b(T * K * D)
    rows = b(T * (H + 2 * K) * D)
    good = dict(plan=plan, positions=pos, dtype="f32", n_tokens=T, head_dim=D, eps=1e-6, n_heads=H, n_kv=K, q=q,
                q_norm=b(D), q_out=qo, k=k, k_norm=b(D), k_out=ko, v=v, slots=slots, k_cache=b(2 * 16 * D),
                v_cache=b(2 * 16 * D), page_size=16, n_pages=2)
    NormRope(ctx, **good)()
    ctx.sync()
    for bad in (dict(n_tokens=0), dict(n_tokens=5), dict(head_dim=7), dict(head_dim=2048), dict(eps=-1.0),
                dict(eps=float("nan")), dict(n_heads=0, n_kv=0), dict(n_heads=3), dict(q_norm=b(D - 1)),
                dict(plan=b(64)), dict(plan=rope_plan(ctx, 16, 1e4)), dict(positions=b(3)), dict(q=None),
                dict(q_out=None), dict(slots=None, k_out=None), dict(v=None), dict(k_cache=None), dict(page_size=0),
                dict(n_pages=3), dict(q_off=1), dict(q_stride=H * D - 1), dict(q_stride=H * D + 1),
                dict(q_out=k), dict(q_out=ko), dict(k_out=v), dict(k_cache=good["v_cache"]),
                dict(q=rows, q_off=D, q_out=rows), dict(q=rows, q_stride=(H + 2 * K) * D, q_out=rows)):
        with pytest.raises(CwError) as e:
            NormRope(ctx, **{**good, **bad})()
        assert e.value.status == 1, bad
    with pytest.raises(ValueError):
        NormRope(ctx, **{**good, "layout": "other"})
    # a slot outside the cache is skipped and reported
    kc = b(2 * 16 * D)
    NormRope(ctx, **{**good, "slots": i32(ctx, [0, 32, 1, 2]), "k_cache": kc})()
    with pytest.raises(CwError) as e:
        ctx.sync()
    assert e.value.status == 1
    ctx.sync()
