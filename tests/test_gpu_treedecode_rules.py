"""Tree decode with penalties, biases and allowed tokens whose prompts are taken in by pieces of a
step: the logits that each token is picked from, against the per-op forward pass."""
import numpy as np
import pytest

import prompt_ref
from test_gpu_promptdecode import teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rules", [dict(penalties=(1.3, 0.4, 0.2)), dict(penalties=(1.2, 0.3, 0.1), biases={11: 3.0},
                                                                          allowed=range(0, 200, 3))])
def test_rules_on_prompts_in_pieces(ctx, tmp_path, rules):
    from chat_wgpu_b200 import gguf
    from chat_wgpu_b200.model import OpByOpQwen3
    from chat_wgpu_b200.treedecode import TreeDecoder
    model = OpByOpQwen3(ctx, gguf.synth_model(str(tmp_path / "m.gguf"), gguf.CONFIGS["tiny-qwen3"], seed=8))
    new, prompts = 8, [[1, 5, 9, 2, 1, 5, 9, 2, 1, 5], list(range(20, 90)), [3]]
    d = TreeDecoder(model, prompts, max_seq=128, chunk=16, **rules)
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
            want, best = prompt_ref.adjust(raw[i][None], "f32", [rules["penalties"]], [s.tokens[:s.n_prompt + i]],
                                           [s.n_prompt], [list(rules["biases"].items())] if "biases" in rules else None,
                                           allow, None if allow is None else [0])
            # the projections' tolerance (1e-3 relative), which a division by at most 1.3 and
            # sums leave as it is; a near tie goes either way
            on = np.isfinite(want[0])
            scale = float(np.sqrt(np.mean(raw[i].astype(np.float64) ** 2)))
            assert np.abs(got[r, i][on] - want[0][on]).max() <= 5e-3 * 1.3 * scale, (r, i)
            top = np.sort(want[0][on])[-2:]
            if top[1] - top[0] > 2e-2 * scale:
                assert s.produced[i] == int(best[0]), (r, i)
    d.close()
    ctx.clear_cache()
