"""The MX8 operators' host side (no GPU): buffer sizes, and arguments refused before any CUDA call."""
import ctypes as ct

import numpy as np
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
    (dict(rows=2 ** 31 - 1, cols=4096, ld=4096, ldv=4096), "too many"),
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


class Fake:
    """Stands for a contiguous CUDA tensor; counts nothing and holds nothing."""

    def __init__(self, shape, dtype="torch.float32", size=4, device=0, stride=None, ptr=P):
        self.shape, self.dtype, self.size, self.device, self.ptr = tuple(shape), DTYPES[dtype], size, device, ptr
        self.strides = stride or tuple(int(np.prod(shape[k + 1:])) for k in range(len(shape)))
        self.nbytes = int(np.prod(shape)) * size

    def stride(self):
        return self.strides

    def is_contiguous(self):
        return self.strides == tuple(int(np.prod(self.shape[k + 1:])) for k in range(len(self.shape)))

    def element_size(self):
        return self.size

    def numel(self):
        return int(np.prod(self.shape))

    def get_device(self):
        return self.device

    def data_ptr(self):
        return self.ptr


class Dtype:
    def __init__(self, name):
        self.name = name

    def __str__(self):
        return self.name


DTYPES = {n: Dtype(n) for n in ("torch.float32", "torch.float16", "torch.bfloat16", "torch.uint8", "torch.int32", "torch.float64")}


def u8(*shape, **other):
    return Fake(shape, "torch.uint8", 1, **other)


def matrix(rows, cols, device=0):
    return mx8.Matrix(u8(rows, (cols + 15) // 16 * 16, device=device), u8(mx8.scale_bytes(rows, cols), device=device), rows, cols)


def test_matrix_reads_its_buffers():
    m = mx8.Matrix(u8(5, 64, stride=(80, 1), ptr=0x2000), u8(512, ptr=0x4000), rows=5, cols=50)
    assert (m.rows, m.cols, m.ld, m.device) == (5, 50, 80, 0)
    assert mx8.Matrix(u8(320), u8(600), 5, 50).ld == 64            # flat bytes
    assert mx8.Matrix(u8(1, 112, stride=(7, 1)), u8(512), 1, 100).ld == 112  # a single row's stride says nothing


@pytest.mark.parametrize("values,scales,rows,cols,word", [
    (u8(5, 48), u8(512), 5, 50, "bytes"), (u8(4, 64), u8(512), 5, 50, "bytes"), (u8(5, 64, 1, stride=(128, 2, 1)), u8(512), 5, 50, "bytes"),
    (u8(5, 64, stride=(64, 2)), u8(512), 5, 50, "bytes"), (Fake((5, 128), size=4, stride=(256, 1)), u8(512), 5, 50, "bytes"),
    (u8(5, 64), u8(511), 5, 50, "scales"), (u8(5, 64), u8(1024, stride=(2,)), 5, 50, "scales"), (u8(5, 64), u8(512, device=1), 5, 50, "CUDA"),
    (u8(5, 64, device=-1), u8(512, device=-1), 5, 50, "CUDA"), (u8(5, 64), u8(512), -1, 50, "shape"), (u8(5, 64), u8(512), 5, 0, "shape"),
    (u8(5, 64), u8(512), 2 ** 40, 50, "range"),
])
def test_matrix_refuses(values, scales, rows, cols, word):
    with pytest.raises(ValueError, match=word):
        mx8.Matrix(values, scales, rows, cols)


@pytest.mark.parametrize("call,word", [
    (lambda: mx8.quantize(Fake((4, 31)), matrix(4, 32)), r"x must be \[4\]\[32\], got \(4, 31\)"),
    (lambda: mx8.quantize(Fake((128,)), matrix(4, 32)), "must be"),
    (lambda: mx8.quantize(Fake((4, 32), "torch.float64", 8), matrix(4, 32)), "float32"),
    (lambda: mx8.quantize(Fake((4, 32), "torch.int32"), matrix(4, 32)), "float32"),
    (lambda: mx8.quantize(Fake((4, 32), device=1), matrix(4, 32)), "device"),
    (lambda: mx8.dequantize(matrix(4, 32), Fake((4, 32), stride=(1, 4))), "contiguous"),
    (lambda: mx8.dequantize(matrix(4, 32), Fake((4, 32), stride=(16, 1))), "stride"),
    (lambda: mx8.dequantize(matrix(4, 32), Fake((4, 32), ptr=P + 2)), "aligned"),
    (lambda: mx8.rms_norm(Fake((4, 32)), Fake((31,)), matrix(4, 32)), "weight"),
    (lambda: mx8.rms_norm(Fake((4, 32)), None, matrix(4, 32)), "weight"),
    (lambda: mx8.rms_norm(Fake((4, 32)), Fake((32,)), matrix(4, 32), eps=-1), "eps"),
    (lambda: mx8.rms_norm(Fake((4, 32)), Fake((32,)), matrix(4, 32), residual=Fake((4, 32)),
                          sum_out=Fake((4, 32), "torch.float16", 2)), "type"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 64), Fake((4, 8))), "columns"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32, device=1), Fake((4, 8))), "device"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32), matrix(4, 9)), "result"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32), Fake((4, 8)), activation="tanh"), "tanh"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32), Fake((4, 8)), activation=3), "activation"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32), Fake((4, 8)), gate=matrix(9, 32)), "gate"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32), Fake((4, 8)), gate_bias=Fake((8,))), "gate"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32), Fake((4, 8)), bias=Fake((8,), "torch.float16", 2)), "bias"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32), Fake((4, 8)), residual=Fake((4, 8), stride=(0, 1))), "stride"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32), Fake((4, 8)), err=Fake((1,))), "err"),
])
def test_calls_refuse(call, word):
    with pytest.raises(ValueError, match=word):
        call()


@pytest.mark.parametrize("call,word", [
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32)), "out"),
    (lambda: mx8.linear(matrix(4, 32), Fake((8, 32)), Fake((4, 8))), "Matrix"),
    (lambda: mx8.linear(matrix(4, 32), matrix(8, 32), Fake((4, 8)), gate=Fake((8, 32))), "Matrix"),
    (lambda: mx8.quantize(Fake((4, 32)), matrix(4, 32), speed=1), "speed"),
    (lambda: mx8.quantize(Fake((4, 32)), matrix(4, 32), out=matrix(4, 32)), "multiple"),
    (lambda: mx8.quantize(Fake((4, 32)), matrix(4, 32), 0, 0), "at most"),
    (lambda: mx8.quantize(Fake((4, 32)), matrix(4, 32), stream="s"), "int"),
    (lambda: mx8.Matrix(u8(5, 64), u8(512), 5), "cols"),
])
def test_calls_refuse_other_types(call, word):
    with pytest.raises(TypeError, match=word):
        call()


def test_a_failing_tensor_attribute_is_passed_on():
    class Broken(Fake):
        def data_ptr(self):
            raise OSError("gone")
    with pytest.raises(OSError, match="gone"):
        mx8.quantize(Broken((4, 32)), matrix(4, 32))
    with pytest.raises(AttributeError):
        mx8.quantize(object(), matrix(4, 32))


def test_tensors_on_the_host_are_refused():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="CUDA"):
        mx8.Matrix.empty(torch.zeros(1), 4, 32)


@pytest.fixture
def calls(monkeypatch):
    """The extension over functions of the test's own in place of the library's: what would have been launched, as
    (name, argument structure, stream), with device 0 the current one."""
    from laya_cuda import _mx8
    made = []

    def entry(name, structure, *more):
        def function(args, *rest):
            kept = structure()
            ct.memmove(ct.byref(kept), args, ct.sizeof(structure))
            made.append((name, kept, rest[-1]))
            return 0
        return ct.CFUNCTYPE(ct.c_int, ct.c_void_p, *more, ct.c_void_p)(function)

    @ct.CFUNCTYPE(ct.c_int, ct.POINTER(ct.c_int))
    def current_device(out):
        out[0] = 0
        return 0

    functions = (entry("quantize", _lib.Mx8Convert), entry("dequantize", _lib.Mx8Convert), entry("rms_norm", _lib.RmsNormMx8),
                 entry("linear", _lib.Mx8Linear, ct.c_void_p), ct.CFUNCTYPE(ct.c_char_p, ct.c_void_p)(lambda e: b""), current_device)
    _mx8.bind(*(ct.cast(f, ct.c_void_p).value for f in functions))
    yield made
    mx8._bind()


def on(device):
    """One call of each operator with everything on `device`."""
    x, m, w = Fake((4, 32), device=device), matrix(4, 32, device), matrix(8, 32, device)
    return (lambda: mx8.quantize(x, m), lambda: mx8.dequantize(m, x), lambda: mx8.rms_norm(x, Fake((32,), device=device), m),
            lambda: mx8.linear(m, w, Fake((4, 8), device=device)))


def test_buffers_on_another_device_than_the_current_one_are_refused(calls):
    for call in on(1):
        with pytest.raises(ValueError, match="on CUDA device 1, the current device is 0"):
            call()
    assert not calls
    for call in on(0):
        call()
    assert [name for name, _, _ in calls] == ["quantize", "dequantize", "rms_norm", "linear"]


def test_current_device(lib):
    device = ct.c_int(7)
    code = lib.laya_current_device(ct.byref(device))
    assert (code == 0 and device.value >= 0) or (code == _lib.ERR_NO_DEVICE and device.value == -1)
    assert lib.laya_current_device(None) == _lib.ERR_INVALID


def test_a_matrix_is_where_its_buffers_are_now(calls):
    """Storage that moved, went to the host or shrank after a Matrix of it was made."""
    m, w = matrix(4, 32), matrix(8, 32)
    m.values.ptr, m.scales.ptr, w.values.ptr, w.scales.ptr = 0x21000, 0x22000, 0x23000, 0x24000
    x, y = Fake((4, 32)), Fake((4, 8))
    mx8.quantize(x, m), mx8.dequantize(m, x), mx8.rms_norm(x, Fake((32,)), m), mx8.linear(m, w, y, gate=w)
    for _, a, _ in calls[:3]:
        assert (a.values, a.scales, a.ldv) == (0x21000, 0x22000, 32)
    a = calls[3][1]
    assert (a.x, a.x_scales, a.w, a.w_scales, a.gate, a.gate_scales) == (0x21000, 0x22000, 0x23000, 0x24000, 0x23000, 0x24000)
    del calls[:]
    m.values.strides = (80, 1)
    assert m.ld == 80
    mx8.quantize(x, m)
    assert calls[0][1].ldv == 80
    del calls[:]
    for change, word in ((dict(device=-1), "CUDA device"), (dict(device=1), "device"), (dict(shape=(3, 32)), "bytes"),
                         (dict(strides=(32, 2)), "bytes")):
        broken = matrix(4, 32)
        for name, value in change.items():
            setattr(broken.values, name, value)
        for call in (lambda: mx8.quantize(x, broken), lambda: mx8.dequantize(broken, x), lambda: mx8.rms_norm(x, Fake((32,)), broken),
                     lambda: mx8.linear(broken, w, y), lambda: mx8.linear(m, broken, Fake((4, 4))),
                     lambda: mx8.linear(m, w, y, gate=broken), lambda: mx8.linear(m, matrix(32, 32), broken), lambda: broken.ld):
            with pytest.raises(ValueError, match=word):
                call()
    small = matrix(4, 32)
    small.scales.shape = (511,)
    small.scales.strides = (1,)
    with pytest.raises(ValueError, match="scales"):
        mx8.quantize(x, small)
    assert not calls


@pytest.mark.parametrize("name", ["laya_op_mx8_quantize", "laya_op_mx8_dequantize"])
@pytest.mark.parametrize("cols", [2 ** 31 - 128, 2 ** 31 - 127, 2 ** 31 - 1])
def test_conversions_refuse_too_many_values_in_the_widest_rows(lib, name, cols):
    with pytest.raises(ValueError, match="too many"):
        _lib.check(getattr(lib, name)(ct.byref(convert(rows=200, cols=cols, ld=cols, ldv=2 ** 31)), None))


@pytest.mark.parametrize("rows,features", [(2 ** 31 - 255, 1), (2 ** 31 - 1, 1), (1, 2 ** 31 - 255), (300, 2 ** 31 - 1)])
def test_linear_refuses_results_whose_tiles_pass_32_bits(lib, rows, features):
    with pytest.raises(ValueError, match="at most 2147483392"):
        _lib.check(lib.laya_op_mx8_linear(ct.byref(linear(rows=rows, features=features, ldo=2 ** 31)), None, None))


class DLTensor(ct.Structure):
    _fields_ = [("data", ct.c_void_p), ("device_type", ct.c_int32), ("device_id", ct.c_int32), ("ndim", ct.c_int32),
                ("code", ct.c_uint8), ("bits", ct.c_uint8), ("lanes", ct.c_uint16), ("shape", ct.POINTER(ct.c_int64)),
                ("strides", ct.POINTER(ct.c_int64)), ("byte_offset", ct.c_uint64)]


class DLExchange(ct.Structure):
    _fields_ = [("major", ct.c_uint32), ("minor", ct.c_uint32), ("previous", ct.c_void_p), ("managed", ct.c_void_p * 3),
                ("tensor_from_object", ct.c_void_p), ("current_stream", ct.c_void_p)]


def exchanging(streams=None):
    """A Fake whose type offers the DLPack exchange table; `streams`: device -> its current stream."""

    @ct.PYFUNCTYPE(ct.c_int, ct.py_object, ct.POINTER(DLTensor))
    def tensor_from_object(o, out):
        n = len(o.shape)
        o.kept = (ct.c_int64 * n)(*o.shape), (ct.c_int64 * n)(*o.strides)
        code, bits = {"torch.float32": (2, 32), "torch.uint8": (1, 8)}[str(o.dtype)]
        out[0] = DLTensor(o.ptr, 2, o.device, n, code, bits, 1, *(ct.cast(k, ct.POINTER(ct.c_int64)) for k in o.kept), 0)
        return 0

    @ct.PYFUNCTYPE(ct.c_int, ct.c_int32, ct.c_int32, ct.POINTER(ct.c_void_p))
    def current_stream(kind, device, out):
        if kind != 2 or device not in streams:
            return -1
        out[0] = streams[device]
        return 0

    address = lambda f: ct.cast(f, ct.c_void_p).value  # noqa: E731
    table = DLExchange(1, 0, None, (ct.c_void_p * 3)(), address(tensor_from_object), address(current_stream) if streams is not None else None)
    new = ct.pythonapi.PyCapsule_New
    new.restype, new.argtypes = ct.py_object, [ct.c_void_p, ct.c_void_p, ct.c_void_p]
    name = ct.create_string_buffer(b"dlpack_exchange_api")
    members = {"__dlpack_c_exchange_api__": new(ct.addressof(table), ct.addressof(name), None),
               "alive": (table, name, tensor_from_object, current_stream)}
    return type("Exchanging", (Fake,), members)


def test_calls_without_a_stream_take_the_frameworks_current_one(calls):
    streams = {0: 0x770}
    cls = exchanging(streams)
    u = lambda *shape: cls(shape, "torch.uint8", 1)  # noqa: E731
    m, w = mx8.Matrix(u(4, 32), u(512), 4, 32), mx8.Matrix(u(8, 32), u(512), 8, 32)
    x = cls((4, 32))

    def each(**how):
        del calls[:]
        mx8.quantize(x, m, **how), mx8.dequantize(m, x, **how)
        mx8.rms_norm(x, cls((32,)), m, **how), mx8.linear(m, w, cls((4, 8)), **how)
        return [stream for _, _, stream in calls]

    assert each() == [0x770] * 4
    assert each(stream=None) == [0x770] * 4
    assert each(stream=0) == [None] * 4  # the legacy default stream
    assert each(stream=0x99) == [0x99] * 4
    streams[0] = 0x880
    assert each() == [0x880] * 4
    streams.clear()
    with pytest.raises(RuntimeError, match="current stream"):
        mx8.quantize(x, m)
    # Types that do not tell.
    cls = exchanging()
    m, w, x = mx8.Matrix(u(4, 32), u(512), 4, 32), mx8.Matrix(u(8, 32), u(512), 8, 32), cls((4, 32))
    assert each() == [None] * 4
    cls = Fake
    m, w, x = matrix(4, 32), matrix(8, 32), Fake((4, 32))
    assert each() == [None] * 4


def test_empty_makes_no_more_bytes_than_the_matrix_has():
    torch = pytest.importorskip("torch")
    asked = []

    class Like(Fake):
        def new_zeros(self, n, dtype=None):
            asked.append((n, dtype))
            made = u8(n)
            made.view = lambda rows, room: u8(rows, room)
            made.byte = lambda: made
            return made

    m = mx8.Matrix.empty(Like((4,)), 300, 50)
    assert (m.rows, m.cols, m.ld, m.values.shape, m.scales.shape) == (300, 50, 64, (300, 64), (3 * 512,))
    assert asked == [(300 * 64, torch.uint8), (3 * 512, torch.uint8)]
    for bad in (object(), Fake((4,))):
        with pytest.raises(AttributeError):
            mx8.Matrix.empty(bad, 4, 32)
