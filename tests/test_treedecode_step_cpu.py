"""What a step of the tree decode builds on the host, without a GPU: no row's whole text unless a
token is picked from the row and its history counts."""
import types

import numpy as np
import pytest


class Text(list):
    """Tokens that count how many of them are copied out."""
    copied = 0

    def __getitem__(self, at):
        got = list.__getitem__(self, at)
        if isinstance(at, slice):
            Text.copied += len(got)
        return got

    def __iter__(self):
        Text.copied += len(self)
        return list.__iter__(self)


class Context:
    def storage(self, a):
        return types.SimpleNamespace(values=np.asarray(a).ravel(), release=lambda: None)

    storage_u32 = storage

    def empty(self, n):
        return None

    def empty_persistent(self, n):
        return self.storage(np.zeros(1))

    def read_u32(self, b, n):
        return np.zeros(n, np.uint32)

    def reset_frame(self):
        pass

    def copy(self, *a):
        pass


def decoder(monkeypatch, prompt, **more):
    from chat_wgpu_b200 import treedecode as td
    monkeypatch.setattr(td.rope, "rope_plan", lambda *a: None)
    monkeypatch.setattr(td.argmax, "argmax", lambda *a: None)
    calls = []

    def adjust(ctx, **kw):
        calls.append(kw)
        return lambda: None

    monkeypatch.setattr(td.rules, "AdjustLogits", adjust)
    model = types.SimpleNamespace(ctx=Context(), n_kv_heads=1, head_dim=8, n_layers=0, rope_theta=1e4, vocab=50)
    d = td.TreeDecoder(model, [prompt], max_seq=4000, draft=lambda tokens: [(-1, 7), (0, 8), (-1, 9)], **more)
    d._forward = lambda rows, *a: rows
    s = d.sessions[0]
    s.tokens = Text(s.tokens)
    return d, s, calls


@pytest.mark.parametrize("rules", [{}, dict(penalties=(1.1, 0.0, 0.0)), dict(biases={3: 1.0})])
def test_pieces_of_a_prompt_copy_their_rows_only(monkeypatch, rules):
    d, s, calls = decoder(monkeypatch, list(range(3000)), **rules)
    s.stored = 2000
    Text.copied = 0
    d.step(5)
    assert s.stored == 2064 and not s.produced
    assert Text.copied <= 2 * 64


def test_picked_rows_have_their_text(monkeypatch):
    """With penalties the last open row and the drafted ones carry their histories; without, no
    row does."""
    d, s, calls = decoder(monkeypatch, [5, 6, 5, 6], penalties=(1.1, 0.0, 0.0))
    s.stored = 1
    d.step(5)
    starts, tokens = calls[0]["starts"].values.view(np.int32), calls[0]["tokens"].values.view(np.int32)
    rows = [tokens[a:b].tolist() for a, b in zip(starts, starts[1:])]
    text = [5, 6, 5, 6]
    assert rows == [[], [], text, text + [7], text + [7, 8], text + [9]]
    assert calls[0]["prompts"].values.tolist() == [4] * 6
    d, s, calls = decoder(monkeypatch, list(range(100)) * 3, biases={3: 1.0})
    s.stored = 299
    Text.copied = 0
    d.step(5)
    assert len(s.produced) >= 1 and "tokens" not in calls[0]
    assert Text.copied <= 20
