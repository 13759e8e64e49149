import ctypes as C

from .. import _lib
from ..context import Buffer


def op(ctx, fn: str, *args) -> Buffer:
    out = C.c_uint64()
    _lib.call(fn, ctx.handle, *args, C.byref(out))
    return Buffer(ctx, out.value)


# element types of the paged operators (CW_GGUF_*)
TYPES = {"f32": 0, "f16": 1, "bf16": 30}


class Prepared:
    """A call whose argument struct is filled once and used every step: calling
    the object enqueues the operator on the context's stream.  It holds its
    buffers; their contents are read when the operator runs."""

    _fn = ""
    _struct = None

    def __init__(self, ctx, **fields):
        self.ctx = ctx
        self.args = self._struct()
        self._keep = []
        for name, value in fields.items():
            if value is None:
                continue
            if isinstance(value, Buffer):
                self._keep.append(value)
                value = value.handle
            setattr(self.args, name, value)
        self._call = getattr(_lib.load(), self._fn)
        self._ref = C.byref(self.args)

    def __call__(self) -> None:
        rc = self._call(self.ctx._h, self._ref)
        if rc:
            _lib.fail(rc, self._fn)


def type_code(dtype: str) -> int:
    if dtype not in TYPES:
        raise ValueError(f"dtype {dtype!r}: one of {sorted(TYPES)}")
    return TYPES[dtype]
