"""Sizes that the tree decode refuses, on the CPU."""
import pytest


def test_chunks_that_cannot_step_are_refused():
    from chat_wgpu_b200.treedecode import TreeDecoder

    class Model:  # refused before the model is used
        ctx = None

    for chunk in (0, -1, 1025):
        with pytest.raises(ValueError, match="chunk"):
            TreeDecoder(Model(), [[1, 2]], max_seq=16, chunk=chunk)
