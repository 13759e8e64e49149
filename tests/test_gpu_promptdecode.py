"""Whole prompts taken in at once and tokens chosen from adjusted logits: the prompt and
logits operators together, against the per-op forward pass."""
import numpy as np
import pytest

import prompt_ref

pytestmark = pytest.mark.gpu


def teacher(ctx, model, tokens, n_prompt):
    """Raw logits that each token behind the prompt is chosen from."""
    ctx.clear_cache()
    cache, out = model.new_cache(len(tokens)), []
    for pos in range(len(tokens) - 1):
        ctx.reset_frame()
        h = model.forward(model.embed(tokens[pos]), pos, cache)
        if pos >= n_prompt - 1:
            out.append(ctx.read(model.logits(h), model.vocab).copy())
    return out


@pytest.mark.parametrize("name,seed,page,rules", [
    ("tiny-qwen3", 7, 16, {}),
    ("small-qwen3", 3, 8, dict(penalties=(1.3, 0.4, 0.2), biases={11: 3.0, 40: -50.0})),
    ("odd-qwen3", 5, 5, dict(penalties=(1.0, 2.0, 1.0), allowed=range(0, 200, 3))),
    ("tiny-qwen3", 9, 16, dict(biases={5: 1.5}))])
def test_prompts_in_and_tokens_out(ctx, tmp_path, name, seed, page, rules):
    from chat_wgpu_b200 import gguf
    from chat_wgpu_b200.model import OpByOpQwen3
    from chat_wgpu_b200.treedecode import TreeDecoder
    path = gguf.synth_model(str(tmp_path / f"{name}.gguf"), gguf.CONFIGS[name], seed=seed)
    model = OpByOpQwen3(ctx, path)
    new = 12
    prompts = [[1, 5, 9, 2, 1, 5, 9, 2, 1, 5], [3], list(range(20, 157)), [7, 8]]
    d = TreeDecoder(model, prompts, max_seq=256, page_size=page, chunk=16, **rules)
    d.prefill()
    assert [s.stored for s in d.sessions] == [9, 0, 136, 1] and d.steps == 0
    d.prefill()  # the one-token prompt has nothing to take in, the others are in
    assert [s.stored for s in d.sessions] == [9, 0, 136, 1]
    got = {}
    while any(len(s.produced) < new for s in d.sessions):
        for s, i, logits in d.step(new, want_logits=True):
            got[d.sessions.index(s), i] = logits
    allow = None
    if "allowed" in rules:
        allow = np.zeros((1, model.vocab), bool)
        allow[0, list(rules["allowed"])] = True
    for r, s in enumerate(d.sessions):
        raw = teacher(ctx, model, s.tokens, s.n_prompt)
        for i in range(new):
            text = s.tokens[:s.n_prompt + i]
            pen = rules.get("penalties")
            want, best = prompt_ref.adjust(
                raw[i][None], "f32", None if pen is None else [pen], [text], [s.n_prompt],
                [list(rules["biases"].items())] if "biases" in rules else None, allow,
                None if allow is None else [0])
            # the projections' tolerance (1e-3 relative, tensor-core GEMM against GEMV), which
            # a division by at most 1 and sums leave as it is; a near tie goes either way
            on = np.isfinite(want[0])
            assert (np.isneginf(got[r, i]) == ~on).all()
            scale = float(np.sqrt(np.mean(raw[i].astype(np.float64) ** 2)))
            assert np.abs(got[r, i][on] - want[0][on]).max() <= 5e-3 * 1.3 * scale, (r, i)
            top = np.sort(want[0][on])[-2:]
            if top[1] - top[0] > 2e-2 * scale:
                assert s.produced[i] == int(best[0]), (r, i)
    d.close()
    ctx.clear_cache()


def test_prefill_gives_the_steps_cache(ctx, tmp_path):
    """The next step's logits after prefill and after a prompt in pieces are the same to the
    projections' tolerance, for prompts longer than a step may be."""
    from chat_wgpu_b200 import gguf
    from chat_wgpu_b200.model import OpByOpQwen3
    from chat_wgpu_b200.treedecode import TreeDecoder
    path = gguf.synth_model(str(tmp_path / "m.gguf"), gguf.CONFIGS["tiny-qwen3"], seed=4)
    model = OpByOpQwen3(ctx, path)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, model.vocab, k).tolist() for k in (700, 90, 333)]
    first = {}
    for way in ("prefill", "pieces"):
        d = TreeDecoder(model, prompts, max_seq=720, chunk=128)
        if way == "prefill":
            d.prefill()
        while any(not s.produced for s in d.sessions):
            for s, i, logits in d.step(1, want_logits=True):
                first[way, d.sessions.index(s)] = logits
        d.close()
    for r in range(3):
        a, b = first["prefill", r], first["pieces", r]
        assert np.abs(a - b).max() <= 5e-3 * float(np.sqrt(np.mean(b.astype(np.float64) ** 2)))
    ctx.clear_cache()
