"""Per-op host wrappers, one module per reference module in chat-wgpu
src/kernels/ (q4, attention, norm, rope, activation, argmax).  Each function
takes a GpuContext plus buffers and dimensions and returns a new arena
buffer, like its Rust counterpart.  pages, tree, prompt, logits, rope.RopeAppend and
rope.NormRope (no Rust counterpart) are prepared calls that write to buffers of the caller."""
from . import (activation, argmax, attention, logits, norm, pages, prompt, q4, rope,  # noqa: F401
               tree)
