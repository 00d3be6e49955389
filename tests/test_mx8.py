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


def convert(**other):
    fields = dict(rows=4, cols=32, dtype=0, values=P, scales=P, ldv=32, data=P, ld=32)
    return _lib.Mx8Convert(**{**fields, **other})


@pytest.mark.parametrize("name", ["laya_op_mx8_quantize", "laya_op_mx8_dequantize"])
@pytest.mark.parametrize("other,word", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "shape"), (dict(cols=0), "shape"),
    (dict(data=None), "null"), (dict(ld=31), "stride"), (dict(data=P + 2), "aligned"), (dict(ldv=40), "16"),
    (dict(cols=48, ld=48), "at least"), (dict(values=P + 8), "16-byte"), (dict(scales=P + 1), "16-byte"),
    (dict(scales=None), "null"), (dict(values=None), "null"),
])
def test_conversions_refuse(lib, name, other, word):
    with pytest.raises(ValueError, match=word):
        _lib.check(getattr(lib, name)(ct.byref(convert(**other)), None))
    with pytest.raises(ValueError, match="null"):
        _lib.check(getattr(lib, name)(None, None))


def norm(**other):
    fields = dict(rows=4, cols=32, dtype=0, residual_dtype=0, x=P, ldx=32, residual=P, ldr=32, sum_out=P, lds=32, weight=P,
                  values=P, scales=P, ldv=32, eps=1e-6)
    return _lib.RmsNormMx8(**{**fields, **other})


@pytest.mark.parametrize("other,word", [
    (dict(dtype=3), "dtype"), (dict(residual_dtype=9), "dtype"), (dict(x=None), "null"), (dict(ldx=31), "stride"),
    (dict(ldr=8), "stride"), (dict(lds=8), "stride"), (dict(residual=P + 2), "aligned"), (dict(weight=None), "null"),
    (dict(weight=P + 4), "16-byte"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(rows=-2), "shape"),
    (dict(ldv=24), "16"), (dict(values=None), "null"),
])
def test_norm_refuses(lib, other, word):
    with pytest.raises(ValueError, match=word):
        _lib.check(lib.laya_op_rms_norm_mx8(ct.byref(norm(**other)), None))
    with pytest.raises(ValueError, match="null"):
        _lib.check(lib.laya_op_rms_norm_mx8(None, None))


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
    for name in ("laya_op_mx8_quantize", "laya_op_mx8_dequantize"):
        assert getattr(lib, name)(ct.byref(convert(rows=0, values=None, scales=None, data=None)), None) == 0
    assert lib.laya_op_rms_norm_mx8(ct.byref(norm(rows=0, x=None, weight=None, values=None)), None) == 0
    assert lib.laya_op_mx8_linear(ct.byref(linear(rows=0, x=None, w=None, out=None)), None, None) == 0


@pytest.mark.parametrize("cls", [_lib.Mx8Convert, _lib.RmsNormMx8, _lib.Mx8Linear])
def test_packed_arguments_are_the_structure(cls):
    values = [k + 1 if kind is not ct.c_float else 0.5 for k, (_, kind) in enumerate(cls._fields_)]
    packed = mx8._packer(cls)(*values)
    filled = cls.from_buffer_copy(packed)
    assert [getattr(filled, name) for name, _ in cls._fields_] == values


def test_tensors_on_the_host_are_refused():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="CUDA"):
        mx8.Matrix.empty(torch.zeros(1), 4, 32)
