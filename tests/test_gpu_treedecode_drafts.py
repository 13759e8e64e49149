"""Drafted nodes are kept: with drafts that hold the model's own continuation a step
produces as many tokens as the drafted path is long."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(ctx, tmp_path_factory):
    from chat_wgpu_b200 import gguf
    from chat_wgpu_b200.model import OpByOpQwen3
    path = str(tmp_path_factory.mktemp("m") / "tiny.gguf")
    return OpByOpQwen3(ctx, gguf.synth_model(path, gguf.CONFIGS["tiny-qwen3"], seed=7))


@pytest.mark.parametrize("wrong_first", [False, True])
def test_drafts_are_kept(ctx, model, wrong_first):
    """wrong_first: a wrong node before each right one, so that the kept path does not lie
    in order in the cache and its tokens are fed again."""
    from chat_wgpu_b200.treedecode import TreeDecoder
    prompts, new, deep = [[1, 5, 9, 2, 7], [3, 4]], 24, 5
    plain = TreeDecoder(model, prompts, max_seq=64, draft=lambda t: [])
    truth = [p + t for p, t in zip(prompts, plain.generate(new))]
    assert plain.steps == new  # a token a step without drafts
    plain.close()

    def draft(tokens):
        full = next(t for t in truth if t[:len(tokens)] == list(tokens))
        nodes, at = [], -1
        for t in full[len(tokens):len(tokens) + deep]:
            if wrong_first:
                nodes.append((at, (t + 1) % model.vocab))
            nodes.append((at, t))
            at = len(nodes) - 1
        return nodes

    d = TreeDecoder(model, prompts, max_seq=64, draft=draft)
    got = d.generate(new)
    assert [p + t for p, t in zip(prompts, got)] == truth
    assert d.steps == new // (deep + 1)  # deep drafted tokens and the one after them
    d.close()
    ctx.clear_cache()

