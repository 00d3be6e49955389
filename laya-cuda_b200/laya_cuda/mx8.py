"""8-bit linear layers: MX8 matrices, the RMS norm that writes them and the product that reads and
writes them (laya_op_mx8_* of include/laya_b200.h).

An MX8 matrix holds E4M3 values and one power-of-two scale per 32 consecutive values of a row;
`Matrix` names its two buffers.  Tensors are torch's, or anything with the attributes of theirs that
csrc/mx8_python.cpp reads (torch itself is not imported); rows must be contiguous, with any row
stride.
The caller owns every buffer.  The calls are enqueued on `stream` (a cudaStream_t as an integer,
0 being the legacy default stream; without it, torch's current stream, or that of whatever framework
the tensors belong to, and the legacy default stream if its tensors do not tell) of the current
device, where the buffers must be.  They allocate nothing and return at once: a tensor used on
another stream than the one that wrote it is the caller's to order.

    x8 = mx8.Matrix.empty(x, *x.shape)                  # buffers beside x
    mx8.rms_norm(h, weight, x8, residual=r, sum_out=r)  # r += h; x8 = norm(r) in 8 bits
    mx8.linear(x8, up, a8, gate=gate, activation="silu")
    mx8.linear(a8, down, r, residual=r)                 # r += a8 down^T
"""
import ctypes as ct

from . import _lib

try:
    from . import _mx8
except ImportError as e:
    raise RuntimeError("laya_cuda/_mx8 for this Python is missing: build it with `python -m laya_cuda.build`") from e

__all__ = ["Matrix", "dequantize", "linear", "quantize", "rms_norm", "scale_bytes"]


def _bind():
    lib = _lib.load()
    _mx8.bind(*(ct.cast(getattr(lib, name), ct.c_void_p).value for name in (
        "laya_op_mx8_quantize", "laya_op_mx8_dequantize", "laya_op_rms_norm_mx8", "laya_op_mx8_linear", "laya_last_error",
        "laya_current_device")))


_mx8.set_loader(_bind)

Matrix, scale_bytes = _mx8.Matrix, _mx8.scale_bytes
quantize, dequantize, rms_norm, linear = _mx8.quantize, _mx8.dequantize, _mx8.rms_norm, _mx8.linear
