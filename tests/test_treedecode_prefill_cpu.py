"""Host side of TreeDecoder.prefill without a GPU: what it holds at a time, what it refuses, and
what it gives back when a launch fails.  The context and the operators are stand-ins."""
import types

import numpy as np
import pytest


class Held:
    def __init__(self, ctx, n):
        self.ctx, self.n = ctx, n
        ctx.live[id(self)] = self

    def release(self):
        del self.ctx.live[id(self)]


class Context:
    """The arena of a context: slot i of a frame is kept until it is asked for in another size."""

    def __init__(self):
        self.slots, self.cursor, self.live, self.most = [], 0, {}, 0

    def empty(self, n):
        if self.cursor == len(self.slots):
            self.slots.append(None)
        if self.slots[self.cursor] is None or self.slots[self.cursor].n != n:
            self.slots[self.cursor] = types.SimpleNamespace(n=n)
        self.cursor += 1
        self.note()
        return self.slots[self.cursor - 1]

    def empty_persistent(self, n):
        b = Held(self, n)
        self.note()
        return b

    def storage_u32(self, a):
        return Held(self, a.size)

    def note(self):
        self.most = max(self.most, sum(s.n for s in self.slots) + sum(b.n for b in self.live.values()))

    def read_u32(self, b, n):
        return np.full(n, -1, np.int32).view(np.uint32)

    def reset_frame(self):
        self.cursor = 0

    def copy(self, *a):
        pass

    def sync(self):
        pass


@pytest.fixture
def decoder(monkeypatch):
    from chat_wgpu_b200 import treedecode as td
    kv, hd = 1, 8
    fails = []

    def call(ctx, **kw):
        def run():
            if fails:
                raise RuntimeError("launch")
        return run

    monkeypatch.setattr(td.norm, "rmsnorm", lambda ctx, x, w, rows, dim, eps: ctx.empty(rows * dim))
    monkeypatch.setattr(td.attention, "add", lambda ctx, a, b, n: ctx.empty(n))
    monkeypatch.setattr(td.activation, "swiglu", lambda ctx, a, b, n: ctx.empty(n))
    monkeypatch.setattr(td.q4, "q4_0_gemm", lambda ctx, a, w, T, i, o: ctx.empty(T * o))
    monkeypatch.setattr(td.rope, "rope_plan", lambda ctx, *a: ctx.empty_persistent(8))
    monkeypatch.setattr(td.pages, "PagePlan", call)
    monkeypatch.setattr(td.rope, "NormRope", call)
    monkeypatch.setattr(td.prompt, "PromptAttention", call)

    def make(prompts, layers=2, max_seq=64, **more):
        dim, hidden = 16, 32
        w = lambda i, o: ("w", i, o)  # noqa: E731
        layer = dict(attn_norm=0, ffn_norm=0, q_norm=0, k_norm=0, wq=w(dim, 2 * kv * hd), wk=w(dim, kv * hd),
                     wv=w(dim, kv * hd), wo=w(2 * kv * hd, dim), gate=w(dim, hidden), up=w(dim, hidden), down=w(hidden, dim))
        model = types.SimpleNamespace(ctx=Context(), n_layers=layers, n_heads=2 * kv, n_kv_heads=kv, head_dim=hd, dim=dim,
                                      hidden=hidden, vocab=50, eps=1e-6, rope_theta=1e4, embed_tbl=0, final_norm=0,
                                      layers=[layer] * layers)
        d = td.TreeDecoder(model, prompts, max_seq=max_seq, **more)
        d.fails = fails
        return d

    return make


def test_activations_of_one_layer_are_held(decoder):
    """What a prefill adds to the decoder's own memory does not grow with the layers."""
    added = []
    for layers in (1, 2, 12):
        d = decoder([[1] * 30, [2] * 11], layers)
        before = sum(b.n for b in d.ctx.live.values())
        d.prefill()
        assert [s.stored for s in d.sessions] == [29, 10]
        added.append(d.ctx.most - before)
        assert sum(b.n for b in d.ctx.live.values()) == before
    assert added[0] == added[1] == added[2]


def test_prompts_past_max_seq_are_refused(decoder):
    d = decoder([[1] * 20, [2] * 65])
    before = dict(d.ctx.live)
    with pytest.raises(ValueError, match="max_seq"):
        d.prefill()
    assert d.ctx.live == before and not d.ctx.slots and [s.stored for s in d.sessions] == [0, 0]
    decoder([[1] * 64]).prefill()


def test_a_failed_launch_leaves_nothing(decoder):
    d = decoder([[1] * 20, [2] * 7])
    before = dict(d.ctx.live)
    place = d._place

    def late(*a):
        at = place(*a)
        d.fails.append(1)
        return at

    d._place = late
    with pytest.raises(RuntimeError, match="launch"):
        d.prefill()
    assert d.ctx.live == before and [s.stored for s in d.sessions] == [0, 0]
    d.fails.clear()
    d._place = place
    d.prefill()
    assert [s.stored for s in d.sessions] == [19, 6]
