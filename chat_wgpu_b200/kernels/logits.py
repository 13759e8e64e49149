"""Penalties, biases and grammar masks on rows of logits (no reference counterpart: it
chooses the largest logit as it is)."""
from .. import _lib
from ..context import Buffer
from ._util import Prepared, type_code


class AdjustLogits(Prepared):
    """Repetition, frequency and presence penalties from each row's history, its biases
    and its mask of allowed tokens, and the argmax of the result (cw_adjust_logits).
    `out` may be `logits` itself; every part but `logits` and `out` may be left out."""

    _fn = "cw_adjust_logits"
    _struct = _lib.AdjustLogitsArgs
    _rows = dict(logits="stride", out=None)
    _floats = ("penalties", "bias_values")

    def __init__(self, ctx, logits: Buffer, out: Buffer, dtype: str, n_rows: int, vocab: int,
                 penalties: Buffer | None = None, tokens: Buffer | None = None,
                 starts: Buffer | None = None, prompts: Buffer | None = None, n_tokens: int = 0,
                 bias_tokens: Buffer | None = None, bias_values: Buffer | None = None,
                 bias_starts: Buffer | None = None, n_bias: int = 0,
                 masks: Buffer | None = None, mask_rows: Buffer | None = None, n_masks: int = 0,
                 best: Buffer | None = None, off: int = 0, stride: int = 0):
        super().__init__(
            ctx, dtype, logits=logits, penalties=penalties, tokens=tokens, starts=starts,
            prompts=prompts, bias_tokens=bias_tokens, bias_values=bias_values,
            bias_starts=bias_starts, masks=masks, mask_rows=mask_rows, out=out, best=best, off=off,
            stride=stride or vocab, type=type_code(dtype), n_rows=n_rows, vocab=vocab,
            n_tokens=n_tokens, n_bias=n_bias, n_masks=n_masks)
