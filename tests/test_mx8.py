"""The MX8 operators' host side (no GPU): buffer sizes, and arguments refused before any CUDA call."""
import ctypes as ct

import pytest

from laya_cuda import _lib, mx8


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("rows,cols", [(0, 1), (1, 1), (128, 128), (129, 128), (128, 129), (1000, 5000), (2 ** 31 - 1, 4096)])
def test_scale_bytes(lib, rows, cols):
    want = -(-rows // 128) * -(-cols // 128) * 512
    assert mx8.scale_bytes(rows, cols) == want == lib.laya_mx8_scale_bytes(rows, cols)


@pytest.mark.parametrize("rows,cols", [(-1, 4), (4, 0), (4, -1)])
def test_scale_bytes_refuses_bad_shapes(lib, rows, cols):
    assert lib.laya_mx8_scale_bytes(rows, cols) == -1
    with pytest.raises(ValueError):
        mx8.scale_bytes(rows, cols)


P = 0x10000  # stands for an aligned device pointer: every call below is refused before it is used


@pytest.mark.parametrize("args,word", [
    ((3, P, 32, 4, 32, P, 32, P, None), "dtype"),
    ((0, P, 32, -1, 32, P, 32, P, None), "shape"),
    ((0, P, 32, 4, 0, P, 32, P, None), "shape"),
    ((0, None, 32, 4, 32, P, 32, P, None), "null"),
    ((0, P, 31, 4, 32, P, 32, P, None), "stride"),
    ((0, P + 2, 32, 4, 32, P, 32, P, None), "aligned"),
    ((0, P, 32, 4, 32, P, 40, P, None), "16"),
    ((0, P, 48, 4, 48, P, 32, P, None), "at least"),
    ((0, P, 32, 4, 32, P + 8, 32, P, None), "16-byte"),
    ((0, P, 32, 4, 32, P, 32, P + 1, None), "16-byte"),
    ((0, P, 32, 4, 32, P, 32, None, None), "null"),
])
def test_quantize_refuses(lib, args, word):
    with pytest.raises(ValueError, match=word):
        _lib.check(lib.laya_op_mx8_quantize(*args))


def test_dequantize_and_norm_refuse(lib):
    for args in ((None, 32, P, 4, 32, 0, P, 32, None), (P, 32, P, 4, 32, 3, P, 32, None), (P, 32, P, 4, 32, 0, P, 16, None)):
        with pytest.raises(ValueError):
            _lib.check(lib.laya_op_mx8_dequantize(*args))
    good = [0, P, 32, 0, P, 32, P, 32, P, 1e-6, 4, 32, P, 32, P, None]
    for at, bad in ((0, 3), (1, None), (3, 9), (5, 8), (7, 8), (8, None), (8, P + 4), (9, -1.0), (9, float("nan")), (10, -2), (13, 24)):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError):
            _lib.check(lib.laya_op_rms_norm_mx8(*args))


def linear(**other):
    fields = dict(rows=4, features=64, cols=32, activation=0, x=P, x_scales=P, ldx=32, w=P, w_scales=P, ldw=32,
                  out=P, ldo=64, out_dtype=0)
    return _lib.Mx8Linear(**{**fields, **other})


@pytest.mark.parametrize("other,word", [
    (dict(rows=-1), "shape"), (dict(features=0), "shape"), (dict(cols=0), "depth"), (dict(activation=4), "activation"),
    (dict(out_dtype=4), "dtype"), (dict(out_dtype=3), "scales"), (dict(x=None), "null"), (dict(x_scales=None), "null"),
    (dict(ldx=31), "stride"), (dict(ldw=16), "stride"), (dict(w=P + 4), "16-byte"), (dict(gate=P, ldg=32), "null"),
    (dict(gate_bias=P), "gate"), (dict(bias=P + 4), "16-byte"), (dict(residual=P, ldr=63), "stride"),
    (dict(residual=P, ldr=64, residual_dtype=3), "dtype"), (dict(out=None), "null"), (dict(ldo=60), "stride"),
    (dict(out=P + 1), "aligned"),
])
def test_linear_refuses(lib, other, word):
    with pytest.raises(ValueError, match=word):
        _lib.check(lib.laya_op_mx8_linear(ct.byref(linear(**other)), None, None))
    with pytest.raises(ValueError, match="null"):
        _lib.check(lib.laya_op_mx8_linear(None, None, None))


def test_no_rows_needs_no_buffers_and_no_device(lib):
    assert lib.laya_op_mx8_quantize(0, None, 32, 0, 32, None, 32, None, None) == 0
    assert lib.laya_op_mx8_dequantize(None, 32, None, 0, 32, 0, None, 32, None) == 0
    assert lib.laya_op_rms_norm_mx8(0, None, 32, 0, None, 0, None, 0, None, 1e-6, 0, 32, None, 32, None, None) == 0
    assert lib.laya_op_mx8_linear(ct.byref(linear(rows=0, x=None, w=None, out=None)), None, None) == 0


def test_tensors_on_the_host_are_refused():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="CUDA"):
        mx8.Matrix.empty(torch.zeros(1), 4, 32)
