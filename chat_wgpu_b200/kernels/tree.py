"""Attention of drafted token trees over a paged cache (no reference counterpart:
its step is one query over one contiguous cache)."""
from .. import _lib
from ..context import Buffer
from ._util import Prepared, type_code


class TreeAttention(Prepared):
    """Every row attends its request's cached tokens and the nodes of its mask
    (cw_tree_attention).  Without a mask node i sees nodes 0..i: a chain, and with
    one node per request plain decode attention."""

    _fn = "cw_tree_attention"
    _struct = _lib.TreeAttnArgs
    _rows = dict(q="q_stride", k_cache=None, v_cache=None, out=None)

    def __init__(self, ctx, q: Buffer, k_cache: Buffer, v_cache: Buffer, table: Buffer,
                 lens: Buffer, starts: Buffer, out: Buffer, dtype: str, n_req: int, n_rows: int,
                 max_nodes: int, n_heads: int, n_kv: int, head_dim: int, page_size: int,
                 n_pages: int, max_pages: int, mask: Buffer | None = None,
                 positions: Buffer | None = None, window: int = 0, softcap: float = 0.0,
                 scale: float = 0.0, q_off: int = 0, q_stride: int = 0):
        super().__init__(
            ctx, dtype, q=q, k_cache=k_cache, v_cache=v_cache, table=table, lens=lens, starts=starts,
            mask=mask, positions=positions, out=out, q_off=q_off,
            q_stride=q_stride or n_heads * head_dim, type=type_code(dtype), n_req=n_req,
            n_rows=n_rows, max_nodes=max_nodes, n_heads=n_heads, n_kv=n_kv, head_dim=head_dim,
            page_size=page_size, n_pages=n_pages, max_pages=max_pages, window=window, scale=scale,
            softcap=softcap)
