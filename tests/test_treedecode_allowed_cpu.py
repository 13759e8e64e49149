"""Sets of allowed tokens that the tree decode refuses, on the CPU: an id outside the vocabulary
would allow another token or none, and of an empty set token 0 would be picked."""
import types

import numpy as np
import pytest


def make(monkeypatch, **more):
    from chat_wgpu_b200 import treedecode as td
    monkeypatch.setattr(td.rope, "rope_plan", lambda *a: None)
    made = []

    def keep(a):
        made.append(np.asarray(a))
        return types.SimpleNamespace(words=made[-1], release=lambda: None)

    ctx = types.SimpleNamespace(empty_persistent=keep, storage_u32=keep)
    model = types.SimpleNamespace(ctx=ctx, n_kv_heads=1, head_dim=8, n_layers=1, rope_theta=1e4, vocab=70)
    try:
        return td.TreeDecoder(model, [[1, 2]], max_seq=16, **more)
    except ValueError:
        assert not made  # refused before anything is allocated
        raise


def test_allowed_tokens_outside_the_vocabulary_are_refused(monkeypatch):
    for bad in ([], [70], [3, -1], [95], [10 ** 9], np.array([-70])):
        with pytest.raises(ValueError, match="allowed"):
            make(monkeypatch, allowed=bad)
    assert make(monkeypatch).mask is None
    for good in ([0], [69, 3, 3], range(0, 70, 7), {5, 64}, np.array([1, 68])):
        bits = np.unpackbits(make(monkeypatch, allowed=good).mask.words.view(np.uint8), bitorder="little")
        assert np.flatnonzero(bits).tolist() == sorted(set(int(t) for t in good))
