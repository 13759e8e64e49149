"""What the prepared calls of the paged operators refuse before they reach the library,
without a GPU."""
import pytest


def wrapped(t):
    from chat_wgpu_b200.context import Buffer
    return Buffer(None, 1, t)


def tree_call(**over):
    import torch
    from chat_wgpu_b200.kernels.tree import TreeAttention
    i = lambda *s: wrapped(torch.zeros(*s, dtype=torch.int32))  # noqa: E731
    x = lambda *s: wrapped(torch.zeros(*s, dtype=torch.bfloat16))  # noqa: E731
    a = dict(q=x(5, 4 * 64), k_cache=x(3, 2, 16, 64), v_cache=x(3, 2, 16, 64), table=i(2, 3), lens=i(2), starts=i(3),
             mask=i(5, 1), positions=i(5), out=x(5, 4 * 64), dtype="bf16", n_req=2, n_rows=5, max_nodes=3, n_heads=4,
             n_kv=2, head_dim=64, page_size=16, n_pages=3, max_pages=3)
    return TreeAttention(None, **{**a, **over})


def rope_call(**over):
    import torch
    from chat_wgpu_b200.kernels.rope import RopeAppend
    i = lambda *s: wrapped(torch.zeros(*s, dtype=torch.int32))  # noqa: E731
    rows = torch.zeros(6, 8 * 32, dtype=torch.float16)
    q, k, v = rows.split([128, 64, 64], dim=1)
    c = wrapped(torch.zeros(2, 2, 16, 32, dtype=torch.float16))
    a = dict(plan=i(4), positions=i(6), dtype="f16", n_tokens=6, n_heads=4, n_kv=2, head_dim=32, q=wrapped(q),
             q_out=wrapped(torch.zeros(6, 128, dtype=torch.float16)), k=wrapped(k), v=wrapped(v), q_stride=256,
             k_stride=256, v_stride=256, slots=i(6), k_cache=c, v_cache=c, page_size=16, n_pages=2)
    return RopeAppend(None, **{**a, **over})


def test_tensors_of_another_type_are_refused():
    import torch
    tree_call()
    tree_call(mask=wrapped(torch.zeros(5, 1, dtype=torch.uint32)))
    rope_call()
    with pytest.raises(ValueError, match="lens: a tensor of int64"):
        tree_call(lens=wrapped(torch.zeros(2, dtype=torch.int64)))
    with pytest.raises(ValueError, match="k_cache: a tensor of bfloat16"):
        tree_call(dtype="f16", q=wrapped(torch.zeros(5, 256, dtype=torch.float16)))
    with pytest.raises(ValueError, match="q_out"):
        rope_call(q_out=wrapped(torch.zeros(6, 128)))
    with pytest.raises(ValueError, match="positions"):
        rope_call(positions=wrapped(torch.zeros(6)))


def test_tensors_that_lie_otherwise_are_refused():
    import torch
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    tree_call(q=wrapped(z(5, 300)[:, :256]), q_stride=300)
    tree_call(q=wrapped(z(5, 4, 64)))
    tree_call(q=wrapped(z(5, 6, 64)[:, :4]), q_stride=384)
    for name, t in (("k_cache", z(3, 16, 2, 64).transpose(1, 2)), ("table", torch.zeros(3, 2, dtype=torch.int32).T),
                    ("q", z(5, 300)[:, :256]),            # rows 300 apart, said to be 256
                    ("q", z(5, 64, 4).transpose(1, 2)), ("out", z(5, 512)[:, ::2]),
                    ("lens", torch.zeros(1, dtype=torch.int32).expand(2))):
        with pytest.raises(ValueError, match=name):
            tree_call(**{name: wrapped(t)})
    with pytest.raises(ValueError, match="k: strides"):
        rope_call(k_stride=64)


def test_numbers_outside_their_fields_are_refused():
    """A struct field keeps the low bits of a number that does not fit: a call of 2^32 + 5
    rows would be one of 5."""
    for bad in (dict(n_rows=2 ** 32 + 5), dict(n_req=-1), dict(window=-2 ** 32), dict(q_off=-8),
                dict(q_off=2 ** 64), dict(max_pages=2.5)):
        with pytest.raises(ValueError, match=next(iter(bad))):
            tree_call(**bad)
    with pytest.raises(ValueError, match="n_tokens"):
        rope_call(n_tokens=2 ** 32 + 6)
    assert tree_call(window=2 ** 32 - 1).args.window == 2 ** 32 - 1  # fits: the library refuses it
