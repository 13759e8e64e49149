import ctypes as C
from numbers import Integral

from .. import _lib
from ..context import Buffer


def op(ctx, fn: str, *args) -> Buffer:
    out = C.c_uint64()
    _lib.call(fn, ctx.handle, *args, C.byref(out))
    return Buffer(ctx, out.value)


# element types of the paged operators (CW_GGUF_*)
TYPES = {"f32": 0, "f16": 1, "bf16": 30}


DTYPES = {"f32": ("float32",), "f16": ("float16",), "bf16": ("bfloat16",)}


def check_tensor(name: str, t, types, row_stride: int | None) -> None:
    """ValueError unless the wrapped tensor's type is one of `types` and it is contiguous,
    or, where rows may be apart, has contiguous rows `row_stride` elements apart."""
    have = str(getattr(t, "dtype", types[0])).rsplit(".", 1)[-1]
    if have not in types:
        raise ValueError(f"{name}: a tensor of {have}, not {' or '.join(types)}")
    shape, strides = [int(d) for d in t.shape], [int(s) for s in t.stride()]

    def dense(shape, strides):
        step = 1
        for d, s in zip(reversed(shape), reversed(strides)):
            if d != 1 and s != step:
                return False
            step *= d
        return True

    if dense(shape, strides):
        return
    if row_stride is None or not dense(shape[1:], strides[1:]) or strides[0] != row_stride:
        raise ValueError(f"{name}: strides {strides} of shape {shape}"
                         + ("" if row_stride is None else f" with rows {row_stride} apart"))


class Prepared:
    """A call whose argument struct is filled once and used every step: calling
    the object enqueues the operator on the context's stream.  It holds its
    buffers; their contents are read when the operator runs.  A wrapped tensor
    (GpuContext.wrap) must be of the operator's type and lie as it reads it."""

    _fn = ""
    _struct = None
    _rows: dict = {}  # buffers of the call's dtype, and the field of their row stride (or None)
    _floats: tuple = ()  # buffers of f32 whatever the call's dtype; all others hold i32

    def __init__(self, ctx, dtype: str | None = None, **fields):
        self.ctx = ctx
        self.args = self._struct()
        self._keep = []
        types = dict(self._struct._fields_)
        for name, value in fields.items():
            if value is None:
                continue
            if isinstance(value, Buffer):
                if value.owner is not None:
                    want = (DTYPES[dtype] if name in self._rows else
                            DTYPES["f32"] if name in self._floats else ("int32", "uint32"))
                    check_tensor(name, value.owner, want, fields.get(self._rows.get(name)))
                self._keep.append(value)
                value = value.handle
            kind = types[name]
            if kind is not C.c_float:
                if not (isinstance(value, Integral) and 0 <= value < 1 << 8 * C.sizeof(kind)):
                    raise ValueError(f"{name}: {value!r} does not fit its field")
                value = int(value)
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
