"""TreeDecoder.prefill on the device holds the activations of one layer, not of all of them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_prefill_memory_does_not_grow_with_layers(tmp_path):
    torch = pytest.importorskip("torch")
    from chat_wgpu_b200 import GpuContext, gguf
    from chat_wgpu_b200.model import OpByOpQwen3
    from chat_wgpu_b200.treedecode import TreeDecoder
    config = gguf.CONFIGS["tiny-qwen3"]
    held = {}
    for layers in (2, 2, 6):  # the first fills the process's scratch pool and loads the kernels
        path = gguf.synth_model(str(tmp_path / f"{layers}.gguf"), {**config, "n_layers": layers}, seed=4)
        with GpuContext(0) as ctx:
            model = OpByOpQwen3(ctx, path)
            prompts = [np.random.default_rng(1).integers(0, model.vocab, 6000).tolist()]
            d = TreeDecoder(model, prompts, max_seq=6016)
            ctx.sync()
            free = torch.cuda.mem_get_info()[0]
            d.prefill()
            held[layers] = free - torch.cuda.mem_get_info()[0]
            d.close()
    # a layer's buffers of 6000 rows are 20 MB and more
    assert abs(held[6] - held[2]) <= 4 << 20
