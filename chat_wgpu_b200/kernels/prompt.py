"""Causal attention of packed prompts (no reference counterpart: its prompt runs one
token at a time)."""
from .. import _lib
from ..context import Buffer
from ._util import Prepared, type_code


class PromptAttention(Prepared):
    """Rows of several requests, packed one after another, attend their own request's keys
    up to themselves (cw_prompt_attention).  With key_starts a request may have more keys
    than rows: the rows are then its last ones, a later piece of a prompt."""

    _fn = "cw_prompt_attention"
    _struct = _lib.PromptAttnArgs
    _rows = dict(q="q_stride", k="k_stride", v="v_stride", out=None)

    def __init__(self, ctx, q: Buffer, k: Buffer, v: Buffer, starts: Buffer, out: Buffer,
                 dtype: str, n_req: int, n_rows: int, n_heads: int, n_kv: int, head_dim: int,
                 key_starts: Buffer | None = None, n_keys: int | None = None, window: int = 0,
                 softcap: float = 0.0, scale: float = 0.0, q_off: int = 0, k_off: int = 0,
                 v_off: int = 0, q_stride: int = 0, k_stride: int = 0, v_stride: int = 0):
        if key_starts is not None and n_keys is None:
            raise ValueError("key_starts: how many key rows there are, n_keys, goes with it")
        kv = n_kv * head_dim
        super().__init__(
            ctx, dtype, q=q, k=k, v=v, starts=starts, key_starts=key_starts, out=out, q_off=q_off,
            k_off=k_off, v_off=v_off, q_stride=q_stride or n_heads * head_dim,
            k_stride=k_stride or kv, v_stride=v_stride or kv, type=type_code(dtype), n_req=n_req,
            n_rows=n_rows, n_keys=n_rows if n_keys is None else n_keys, n_heads=n_heads,
            n_kv=n_kv, head_dim=head_dim, window=window, scale=scale, softcap=softcap)
