"""Between a layer's projections: rotary positions, and attention over packed sequences with caps, biases by distance
and masks (laya_op_rotary and laya_op_attend of include/laya_b200.h).

Tensors are [tokens][heads][head_dim] with token and head strides of their own, so slices of a projection's result
serve as they are (q, k and v may not be broadcast, and heads that are written may not overlap); they are torch's, or anything with the attributes of theirs that csrc/python_tensors.h
reads (torch itself is not imported).  The caller owns every buffer.  The calls are enqueued on `stream` (a
cudaStream_t as an integer, 0 being the legacy default stream; without it, torch's current stream, or that of
whatever framework the tensors belong to, and the legacy default stream if its tensors do not tell) of the
current device, where the buffers must be.  They allocate nothing and return at once: a tensor used on another
stream than the one that wrote it is the caller's to order.

    qkv = projected.view(tokens, heads + 2 * kv_heads, head_dim)
    q, k, v = qkv[:, :heads], qkv[:, heads:-kv_heads], qkv[:, -kv_heads:]
    attention.rotary(q, positions, q, k=k, k_out=k)                      # in place
    attention.attend(q, k, v, out, starts, lengths, max_queries=longest, max_keys=longest, causal=True, cap=50.0)

`examples/attention_layer.py` runs them between two products of laya_cuda.mx8.
"""
import ctypes as ct

from . import _lib

try:
    from . import _mx8
except ImportError as e:
    raise RuntimeError("laya_cuda/_mx8 for this Python is missing: build it with `python -m laya_cuda.build`") from e

__all__ = ["attend", "rotary"]


def _bind():
    lib = _lib.load()
    _mx8.bind_attention(*(ct.cast(getattr(lib, name), ct.c_void_p).value for name in (
        "laya_op_rotary", "laya_op_attend", "laya_last_error", "laya_current_device")))


_mx8.set_attention_loader(_bind)

rotary, attend = _mx8.rotary, _mx8.attend
