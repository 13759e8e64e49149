"""rope::rope (chat-wgpu src/kernels/rope.rs), and the rotary positions of many
rows at once with k and v written to a paged cache (no reference counterpart)."""
import ctypes as C

from .. import _lib
from ..context import Buffer
from ._util import Prepared, op, type_code


def rope(ctx, x: Buffer, rows: int, head_dim: int, pos: int, theta: float) -> Buffer:
    """Rotate-half RoPE of rows x head_dim at position pos (rope.rs:8-27)."""
    return op(ctx, "cw_rope", x.handle, int(rows), int(head_dim), int(pos), float(theta))


SCALINGS = {"none": 0, "linear": 1, "banded": 2, "yarn": 3}
LAYOUTS = {"half": 0, "interleaved": 1}


def rope_plan(ctx, rot_dim: int, theta: float, kind: str = "none", factor: float = 1.0,
              low: float = 1.0, high: float = 32.0, trained: int = 0,
              amplitude: float = 0.0) -> Buffer:
    """The rotary frequencies of rot_dim elements as a persistent buffer
    (cw_rope_plan): kind none, linear, banded or yarn."""
    sc = _lib.RopeScaling(SCALINGS[kind], int(trained), float(factor), float(low), float(high),
                          float(amplitude))
    b = C.c_uint64()
    _lib.call("cw_rope_plan", ctx.handle, int(rot_dim), float(theta), C.byref(sc), C.byref(b))
    return Buffer(ctx, b.value)


class RopeAppend(Prepared):
    """Rotate a step's q and k rows at their positions and write k and v to their
    cache slots (cw_rope_append).  Without q or without k and v the other half
    alone; strides and offsets count elements (0 = contiguous rows)."""

    _fn = "cw_rope_append"
    _struct = _lib.RopeAppendArgs
    _rows = dict(q="q_stride", k="k_stride", v="v_stride", q_out=None, k_cache=None, v_cache=None)

    def __init__(self, ctx, plan: Buffer, positions: Buffer, dtype: str, n_tokens: int,
                 head_dim: int, layout: str = "half", n_heads: int = 0, n_kv: int = 0,
                 q: Buffer | None = None, q_out: Buffer | None = None, k: Buffer | None = None,
                 v: Buffer | None = None, slots: Buffer | None = None,
                 k_cache: Buffer | None = None, v_cache: Buffer | None = None, page_size: int = 0,
                 n_pages: int = 0, q_off: int = 0, k_off: int = 0, v_off: int = 0,
                 q_stride: int = 0, k_stride: int = 0, v_stride: int = 0):
        if layout not in LAYOUTS:
            raise ValueError(f"layout {layout!r}: one of {sorted(LAYOUTS)}")
        kv = n_kv * head_dim
        super().__init__(
            ctx, dtype, plan=plan, positions=positions, q=q, k=k, v=v, slots=slots, q_out=q_out,
            k_cache=k_cache, v_cache=v_cache, q_off=q_off, k_off=k_off, v_off=v_off,
            q_stride=q_stride or n_heads * head_dim, k_stride=k_stride or kv,
            v_stride=v_stride or kv, type=type_code(dtype), layout=LAYOUTS[layout],
            n_tokens=n_tokens, n_heads=n_heads, n_kv=n_kv, head_dim=head_dim, page_size=page_size,
            n_pages=n_pages)
