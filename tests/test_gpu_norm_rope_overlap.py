"""Head norms with keys and values that are the same rows: right into buffers of their own,
refused in place, where one head's result would be another's input."""
import numpy as np
import pytest

import paged_ref as ref
import prompt_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_shared_keys_and_values(ctx, dtype):
    from chat_wgpu_b200 import CwError
    from chat_wgpu_b200.kernels.rope import NormRope, rope_plan
    T, H, K, D, page = 150, 2, 2, 64, 16
    rng = np.random.default_rng(1)
    x = ref.rounded(rng.normal(0, 1, (T, K * D)), dtype)
    w = rng.normal(1, 0.2, D).astype(np.float32)
    pos = np.arange(T)
    i32 = lambda a: ctx.storage_u32(np.ascontiguousarray(a, np.int32).view(np.uint32))  # noqa: E731
    new = lambda n: ref.upload(ctx, np.zeros(n), dtype)  # noqa: E731
    pages = -(-T // page)
    rows, q, q_out, k_out = ref.upload(ctx, x, dtype), ref.upload(ctx, x, dtype), new(T * H * D), new(T * K * D)
    kc, vc = new(pages * K * page * D), new(pages * K * page * D)
    call = dict(plan=rope_plan(ctx, D, 1e4), positions=i32(pos), dtype=dtype, n_tokens=T, head_dim=D, eps=1e-6, n_heads=H,
                n_kv=K, q=q, q_norm=ctx.storage(w), q_out=q_out, k=rows, k_norm=ctx.storage(w), k_out=k_out, v=rows,
                slots=i32(pos), k_cache=kc, v_cache=vc, page_size=page, n_pages=pages)
    for bad in (dict(k_out=rows), dict(k=q, q_out=q), dict(v=q, q_out=q), dict(q=rows, k_out=rows, v=q)):
        with pytest.raises(CwError) as e:
            NormRope(ctx, **{**call, **bad})()
        assert e.value.status == 1, bad
    NormRope(ctx, **call)()
    ctx.sync()
    f, amp = ref.rates(D, 1e4)
    want = prompt_ref.norm_rotate(x.reshape(T, K, D), w, False, 1e-6, pos, f, amp, "half")
    # norm and rotation below 2^-18 of the head's largest pair, one rounding to the type
    tol = 2.0 ** -18 * 2 * np.abs(want).max(-1, keepdims=True) + ref.UNIT[dtype] * np.abs(want)
    got = ref.read(ctx, k_out, dtype, (T, K, D))
    assert (np.abs(got - want) <= tol).all()
    cached = ref.read(ctx, vc, dtype, (pages, K, page, D)).transpose(0, 2, 1, 3).reshape(-1, K * D)[:T]
    assert np.array_equal(cached, x)
    cached = ref.read(ctx, kc, dtype, (pages, K, page, D)).transpose(0, 2, 1, 3).reshape(-1, K, D)[:T]
    assert np.array_equal(cached, got)
