"""8-bit linear layers: MX8 matrices, the RMS norm that writes them and the product that reads and
writes them (laya_op_mx8_* of include/laya_b200.h).

An MX8 matrix holds E4M3 values and one power-of-two scale per 32 consecutive values of a row;
`Matrix` names its two buffers.  Tensors are anything with torch's `data_ptr`, `shape`, `stride`,
`dtype` and `device` (torch itself is not imported); rows must be contiguous, with any row stride.
The caller owns every buffer.  The calls are enqueued on `stream` (a cudaStream_t as an integer;
0, the default, is the legacy default stream) of the current device, allocate nothing and return
at once: a tensor used on another stream than the one that wrote it is the caller's to order.

    x8 = mx8.Matrix.empty(x, *x.shape)                  # buffers beside x
    mx8.rms_norm(h, weight, x8, residual=r, sum_out=r)  # r += h; x8 = norm(r) in 8 bits
    mx8.linear(x8, up, a8, gate=gate, activation="silu")
    mx8.linear(a8, down, r, residual=r)                 # r += a8 down^T
"""
import ctypes as ct

from . import _lib

ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU, "silu": _lib.ACT_SILU}
_NAMES = {"torch.float32": _lib.DTYPE_F32, "torch.float16": _lib.DTYPE_F16, "torch.bfloat16": _lib.DTYPE_BF16}
_codes = {}  # dtype object -> LAYA_DTYPE_* (None: not one of the three)


def _code(dtype):
    try:
        return _codes[dtype]
    except KeyError:
        return _codes.setdefault(dtype, _NAMES.get(str(dtype)))


def scale_bytes(rows, cols):
    """Bytes of the scales of an MX8 matrix (tiles of 128 rows x 128 columns, 512 bytes each)."""
    if rows < 0 or cols < 1:
        raise ValueError(f"bad shape {rows} x {cols}: rows may be 0, columns may not")
    return -(-rows // 128) * -(-cols // 128) * 512


class Matrix:
    """An MX8 matrix [rows][cols]: `values`, one byte each, [rows][a multiple of 16 of at least
    cols], and `scales`, `scale_bytes(rows, cols)` bytes.  Holds references to both buffers."""

    __slots__ = ("values", "scales", "rows", "cols", "ld", "device", "values_ptr", "scales_ptr")

    def __init__(self, values, scales, rows, cols):
        shape, stride = values.shape, values.stride()
        if len(shape) != 2 or shape[0] != rows or stride[1] != 1 or values.element_size() != 1:
            raise ValueError(f"values of a {rows} x {cols} matrix must be bytes in {rows} contiguous rows, got {tuple(shape)}")
        if scales.element_size() != 1 or scales.numel() < scale_bytes(rows, cols) or not scales.is_contiguous():
            raise ValueError(f"scales of a {rows} x {cols} matrix need {scale_bytes(rows, cols)} contiguous bytes")
        device = values.device
        if device.type != "cuda" or scales.device != device:
            raise ValueError("values and scales must be on the same CUDA device")
        self.values, self.scales, self.rows, self.cols = values, scales, rows, cols
        room = (cols + 15) // 16 * 16
        if shape[1] < room:
            raise ValueError(f"rows of {cols} values need room for {room}, got {shape[1]}")
        self.ld = stride[0] if rows > 1 else room  # the stride of a single row says nothing
        self.device = device
        self.values_ptr, self.scales_ptr = values.data_ptr(), scales.data_ptr()

    @classmethod
    def empty(cls, like, rows, cols):
        """Buffers for a matrix on the device of the torch tensor `like` (uint8, cleared)."""
        byte = like.new_zeros(0).byte().dtype
        return cls(like.new_zeros((rows, (cols + 15) // 16 * 16), dtype=byte),
                   like.new_zeros(scale_bytes(rows, cols), dtype=byte), rows, cols)


def _rows(name, t, rows, cols, device):
    """(pointer, row stride, dtype code) of a [rows][cols] tensor with contiguous rows."""
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows or shape[1] != cols:
        raise ValueError(f"{name} must be [{rows}][{cols}], got {tuple(shape)}")
    stride = t.stride()
    if cols > 1 and stride[1] != 1:
        raise ValueError(f"{name}: the values of a row must be contiguous")
    code = _code(t.dtype)
    if code is None:
        raise ValueError(f"{name}: {t.dtype} is not float32, float16 or bfloat16")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the matrix on {device}")
    return t.data_ptr(), stride[0] if rows > 1 else cols, code


def _vector(name, t, n, device):
    if t is None:
        return None
    if tuple(t.shape) != (n,) or _code(t.dtype) != _lib.DTYPE_F32 or (n > 1 and t.stride(0) != 1) or t.device != device:
        raise ValueError(f"{name} must be {n} contiguous float32 values on {device}")
    return t.data_ptr()


def quantize(x, out, stream=0):
    """x [rows][cols] in 16 or 32 bits -> the Matrix `out`."""
    ptr, ld, code = _rows("x", x, out.rows, out.cols, out.device)
    _lib.check(_lib.load().laya_op_mx8_quantize(code, ptr, ld, out.rows, out.cols, out.values_ptr, out.ld, out.scales_ptr,
                                                stream))


def dequantize(x, out, stream=0):
    """The Matrix `x` -> out [rows][cols] in 16 or 32 bits."""
    ptr, ld, code = _rows("out", out, x.rows, x.cols, x.device)
    _lib.check(_lib.load().laya_op_mx8_dequantize(x.values_ptr, x.ld, x.scales_ptr, x.rows, x.cols, code, ptr, ld, stream))


def rms_norm(x, weight, out, residual=None, sum_out=None, eps=1e-6, stream=0):
    """h = x + residual; sum_out = h; out = h / sqrt(mean(h^2) + eps) * weight, in MX8.

    `residual` and `sum_out` are optional, of one type, and may be the same tensor."""
    rows, cols, device = out.rows, out.cols, out.device
    ptr, ld, code = _rows("x", x, rows, cols, device)
    rptr = sptr = None
    ldr = lds = 0
    rcode = scode = code
    if residual is not None:
        rptr, ldr, rcode = _rows("residual", residual, rows, cols, device)
    if sum_out is not None:
        sptr, lds, scode = _rows("sum_out", sum_out, rows, cols, device)
        if residual is None:
            rcode = scode
        elif scode != rcode:
            raise ValueError("sum_out must have the residual's type")
    _lib.check(_lib.load().laya_op_rms_norm_mx8(code, ptr, ld, rcode, rptr, ldr, sptr, lds,
                                                _vector("weight", weight, cols, device), eps, rows, cols,
                                                out.values_ptr, out.ld, out.scales_ptr, stream))


def linear(x, w, out, bias=None, gate=None, gate_bias=None, activation="none", residual=None, err=None, stream=0):
    """out = act(x w^T + bias) + residual, or, with a `gate` matrix,
    out = act(x gate^T + gate_bias) * (x w^T + bias) + residual.

    x: Matrix [rows][cols]; w, gate: Matrix [features][cols]; out: a Matrix or a tensor
    [rows][features].  bias, gate_bias: float32 [features].  residual: [rows][features] in 16 or 32
    bits, added before the one rounding; it may be `out` itself.  activation: one of ACTIVATIONS.
    err: an int32 tensor, zero on entry, that receives a device error."""
    rows, cols, n, device = x.rows, x.cols, w.rows, x.device
    if w.cols != cols or w.device != device:
        raise ValueError(f"w is {n} x {w.cols} on {w.device}, x has {cols} columns on {device}")
    try:
        act = ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"activation {activation!r} is not one of {sorted(ACTIVATIONS)}") from None
    gptr = gsptr = None
    ldg = 0
    if gate is not None:
        if gate.rows != n or gate.cols != cols or gate.device != device:
            raise ValueError(f"gate is {gate.rows} x {gate.cols}, w {n} x {cols}")
        gptr, gsptr, ldg = gate.values_ptr, gate.scales_ptr, gate.ld
    rptr, ldr, rcode = (None, 0, 0) if residual is None else _rows("residual", residual, rows, n, device)
    if isinstance(out, Matrix):
        if out.rows != rows or out.cols != n or out.device != device:
            raise ValueError(f"out is {out.rows} x {out.cols}, the result {rows} x {n}")
        optr, osptr, ldo, ocode = out.values_ptr, out.scales_ptr, out.ld, _lib.DTYPE_MX8
    else:
        optr, ldo, ocode = _rows("out", out, rows, n, device)
        osptr = None
    if err is not None and (str(err.dtype) != "torch.int32" or err.device != device or err.numel() < 1):
        raise ValueError(f"err must be int32 on {device}")
    args = _lib.Mx8Linear(rows, n, cols, act, x.values_ptr, x.scales_ptr, x.ld, w.values_ptr, w.scales_ptr, w.ld,
                          gptr, gsptr, ldg, _vector("bias", bias, n, device), _vector("gate_bias", gate_bias, n, device),
                          rptr, ldr, optr, osptr, ldo, rcode, ocode)
    _lib.check(_lib.load().laya_op_mx8_linear(ct.byref(args), None if err is None else err.data_ptr(), stream))
