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
import struct

from . import _lib

ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU, "silu": _lib.ACT_SILU}
_NAMES = {"torch.float32": _lib.DTYPE_F32, "torch.float16": _lib.DTYPE_F16, "torch.bfloat16": _lib.DTYPE_BF16}
_codes = {}  # dtype object -> LAYA_DTYPE_* (None: not one of the three)


def _packer(cls):
    """Packs a C argument structure from its fields' values in order (pointers as integers, 0 for NULL).
    A single-token call takes a few microseconds in all, and packed bytes cost a fifth of what ctypes
    spends on the same structure or on as many arguments."""
    letters = {ct.c_int32: "i", ct.c_int64: "q", ct.c_void_p: "P", ct.c_float: "f"}
    packer = struct.Struct("@" + "".join(letters[kind] for _, kind in cls._fields_) + "0P")
    assert packer.size == ct.sizeof(cls)
    return packer.pack


_convert, _norm, _linear = _packer(_lib.Mx8Convert), _packer(_lib.RmsNormMx8), _packer(_lib.Mx8Linear)


def _code(dtype):
    try:
        return _codes[dtype]
    except KeyError:
        return _codes.setdefault(dtype, _NAMES.get(str(dtype)))


def scale_bytes(rows, cols):
    """Bytes of the scales of an MX8 matrix (tiles of 128 rows x 128 columns, 512 bytes each)."""
    if rows < 0 or cols < 1:
        raise ValueError(f"bad shape {rows} x {cols}: rows may be 0, columns may not")
    return (rows + 127 >> 7) * (cols + 127 >> 7) * 512


class Matrix:
    """An MX8 matrix [rows][cols]: `values`, bytes in `rows` rows of cols rounded up to a multiple of
    16, and `scales`, `scale_bytes(rows, cols)` bytes.  Both are contiguous, of any type of that many
    bytes; two-dimensional values of one-byte elements may have a larger row stride.  Holds
    references to both buffers."""

    __slots__ = ("values", "scales", "rows", "cols", "ld", "device", "values_ptr", "scales_ptr")

    def __init__(self, values, scales, rows, cols):
        room = cols + 15 & -16
        if not (values.is_contiguous() and values.nbytes == rows * room):
            shape = values.shape
            if len(shape) != 2 or shape[0] != rows or values.stride(1) != 1 or values.element_size() != 1:
                raise ValueError(f"values of a {rows} x {cols} matrix must be bytes in {rows} contiguous rows, got {tuple(shape)}")
            if shape[1] < room:
                raise ValueError(f"rows of {cols} values need room for {room}, got {shape[1]}")
            self.ld = values.stride(0) if rows > 1 else room  # the stride of a single row says nothing
        else:
            self.ld = room
        if scales.nbytes < scale_bytes(rows, cols) or not scales.is_contiguous():
            raise ValueError(f"scales of a {rows} x {cols} matrix need {scale_bytes(rows, cols)} contiguous bytes")
        self.device = device = values.get_device()
        if device < 0 or scales.get_device() != device:
            raise ValueError("values and scales must be on the same CUDA device")
        self.values, self.scales, self.rows, self.cols = values, scales, rows, cols
        self.values_ptr, self.scales_ptr = values.data_ptr(), scales.data_ptr()

    @classmethod
    def empty(cls, like, rows, cols):
        """Buffers for a matrix on the device of the torch tensor `like` (uint8, cleared)."""
        byte = like.new_zeros(0).byte().dtype
        return cls(like.new_zeros((rows, cols + 15 & -16), dtype=byte),
                   like.new_zeros(scale_bytes(rows, cols), dtype=byte), rows, cols)


def _rows(name, t, rows, cols, device):
    """(pointer, row stride, dtype code) of a [rows][cols] tensor with contiguous rows."""
    if t.shape != (rows, cols):
        raise ValueError(f"{name} must be [{rows}][{cols}], got {tuple(t.shape)}")
    ld = cols
    if not t.is_contiguous():
        if cols > 1 and t.stride(1) != 1:
            raise ValueError(f"{name}: the values of a row must be contiguous")
        if rows > 1:
            ld = t.stride(0)
    code = _code(t.dtype)
    if code is None:
        raise ValueError(f"{name}: {t.dtype} is not float32, float16 or bfloat16")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, the matrix on CUDA device {device}")
    return t.data_ptr(), ld, code


def _vector(name, t, n, device):
    if t.shape != (n,) or _code(t.dtype) != _lib.DTYPE_F32 or not t.is_contiguous() or t.get_device() != device:
        raise ValueError(f"{name} must be {n} contiguous float32 values on CUDA device {device}")
    return t.data_ptr()


def quantize(x, out, stream=0):
    """x [rows][cols] in 16 or 32 bits -> the Matrix `out`."""
    rows, cols = out.rows, out.cols
    ptr, ld, code = _rows("x", x, rows, cols, out.device)
    status = _lib.load().laya_op_mx8_quantize(
        _convert(rows, cols, code, out.values_ptr, out.scales_ptr, out.ld, ptr, ld), stream)
    if status:
        _lib.check(status)


def dequantize(x, out, stream=0):
    """The Matrix `x` -> out [rows][cols] in 16 or 32 bits."""
    rows, cols = x.rows, x.cols
    ptr, ld, code = _rows("out", out, rows, cols, x.device)
    status = _lib.load().laya_op_mx8_dequantize(
        _convert(rows, cols, code, x.values_ptr, x.scales_ptr, x.ld, ptr, ld), stream)
    if status:
        _lib.check(status)


def rms_norm(x, weight, out, residual=None, sum_out=None, eps=1e-6, stream=0):
    """h = x + residual; sum_out = h; out = h / sqrt(mean(h^2) + eps) * weight, in MX8.

    `residual` and `sum_out` are optional, of one type, and may be the same tensor."""
    rows, cols, device = out.rows, out.cols, out.device
    ptr, ld, code = _rows("x", x, rows, cols, device)
    rptr = ldr = sptr = lds = 0
    rcode = code
    if residual is not None:
        rptr, ldr, rcode = _rows("residual", residual, rows, cols, device)
    if sum_out is not None:
        sptr, lds, scode = _rows("sum_out", sum_out, rows, cols, device)
        if residual is None:
            rcode = scode
        elif scode != rcode:
            raise ValueError("sum_out must have the residual's type")
    status = _lib.load().laya_op_rms_norm_mx8(
        _norm(rows, cols, code, rcode, ptr, ld, rptr, ldr, sptr, lds, _vector("weight", weight, cols, device),
              out.values_ptr, out.scales_ptr, out.ld, eps), stream)
    if status:
        _lib.check(status)


def linear(x, w, out, bias=None, gate=None, gate_bias=None, activation="none", residual=None, err=None, stream=0):
    """out = act(x w^T + bias) + residual, or, with a `gate` matrix,
    out = act(x gate^T + gate_bias) * (x w^T + bias) + residual.

    x: Matrix [rows][cols]; w, gate: Matrix [features][cols]; out: a Matrix or a tensor
    [rows][features].  bias, gate_bias: float32 [features].  residual: [rows][features] in 16 or 32
    bits, added before the one rounding; it may be `out` itself.  activation: one of ACTIVATIONS.
    err: an int32 tensor, zero on entry, that receives a device error."""
    rows, cols, n, device = x.rows, x.cols, w.rows, x.device
    if w.cols != cols or w.device != device:
        raise ValueError(f"w is {n} x {w.cols} on device {w.device}, x has {cols} columns on device {device}")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation {activation!r} is not one of {sorted(ACTIVATIONS)}")
    gptr = gsptr = ldg = rptr = ldr = rcode = osptr = bptr = gbptr = eptr = 0
    if gate is not None:
        if gate.rows != n or gate.cols != cols or gate.device != device:
            raise ValueError(f"gate is {gate.rows} x {gate.cols}, w {n} x {cols}")
        gptr, gsptr, ldg = gate.values_ptr, gate.scales_ptr, gate.ld
    if bias is not None:
        bptr = _vector("bias", bias, n, device)
    if gate_bias is not None:
        gbptr = _vector("gate_bias", gate_bias, n, device)
    if residual is not None:
        rptr, ldr, rcode = _rows("residual", residual, rows, n, device)
    if isinstance(out, Matrix):
        if out.rows != rows or out.cols != n or out.device != device:
            raise ValueError(f"out is {out.rows} x {out.cols}, the result {rows} x {n}")
        optr, osptr, ldo, ocode = out.values_ptr, out.scales_ptr, out.ld, _lib.DTYPE_MX8
    else:
        optr, ldo, ocode = _rows("out", out, rows, n, device)
    if err is not None:
        if str(err.dtype) != "torch.int32" or err.get_device() != device or err.numel() < 1:
            raise ValueError(f"err must be int32 on CUDA device {device}")
        eptr = err.data_ptr()
    status = _lib.load().laya_op_mx8_linear(
        _linear(rows, n, cols, act, x.values_ptr, x.scales_ptr, x.ld, w.values_ptr, w.scales_ptr, w.ld,
                gptr, gsptr, ldg, bptr, gbptr, rptr, ldr, optr, osptr, ldo, rcode, ocode), eptr, stream)
    if status:
        _lib.check(status)
