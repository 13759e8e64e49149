"""Greedy decode with drafted trees over a paged cache: the tokens and logits of
plain greedy decode, in fewer steps."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,seed,page,chunk", [("tiny-qwen3", 7, 16, 64), ("small-qwen3", 3, 8, 9),
                                                  ("odd-qwen3", 5, 5, 16)])
def test_tree_decode_equals_greedy(ctx, tmp_path, name, seed, page, chunk):
    from chat_wgpu_b200 import gguf
    from chat_wgpu_b200.model import OpByOpQwen3, generate_op_by_op
    from chat_wgpu_b200.treedecode import TreeDecoder
    path = gguf.synth_model(str(tmp_path / f"{name}.gguf"), gguf.CONFIGS[name], seed=seed)
    model = OpByOpQwen3(ctx, path)
    new = 24
    prompts = [[1, 5, 9, 2, 1, 5, 9, 2, 1, 5], [3], list(range(20, 57))]
    plain = [generate_op_by_op(ctx, model, p, new, want_logits=True) for p in prompts]
    d = TreeDecoder(model, prompts, max_seq=64, page_size=page, chunk=chunk)
    got = {}
    while any(len(s.produced) < new for s in d.sessions):
        for s, i, logits in d.step(new, want_logits=True):
            got[d.sessions.index(s), i] = logits
    for r, (tokens, logits) in enumerate(plain):
        # the projections' tolerance (1e-3 relative, tensor-core GEMM against GEMV) decides
        # a near tie either way: compare up to the first one
        for i in range(new):
            top = np.sort(logits[i])[-2:]
            scale = float(np.sqrt(np.mean(logits[i].astype(np.float64) ** 2)))
            assert np.abs(got[r, i] - logits[i]).max() <= 5e-3 * scale, (r, i)
            if top[1] - top[0] < 1e-2 * scale:
                break
            assert d.sessions[r].produced[i] == int(tokens[i]), (r, i)
    assert d.steps < len(max(prompts, key=len)) + new
    d.close()
    ctx.clear_cache()
