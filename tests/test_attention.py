"""Rotary positions and attention, host side (no GPU): arguments refused before any CUDA call."""
import ctypes as ct

import numpy as np
import pytest

from laya_cuda import _lib, attention


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


P = 0x10000  # stands for an aligned device pointer: every call below is refused before it is used


def rotary(part=None, **other):
    fields = dict(tokens=4, head_dim=64, dims=64, dtype=2, positions=P, theta=10000.0, factor=1.0, length=4096.0, low=1.0, high=32.0,
                  magnitude=1.0)
    args = _lib.Rotary(**{**fields, **other})
    args.part[0] = _lib.Heads(**{**dict(x=P, x_token=128, x_head=64, out=2 * P, out_token=128, out_head=64, heads=2), **(part or {})})
    return args


@pytest.mark.parametrize("other,part,word", [
    (dict(tokens=-1), None, "shape"), (dict(head_dim=0), None, "shape"), (dict(dims=0), None, "dims"), (dict(dims=7), None, "dims"),
    (dict(dims=66), None, "dims"), (dict(head_dim=2000, dims=514), None, "dims"), (dict(dtype=3), None, "dtype"),
    (dict(scaling=4), None, "scaling"), (dict(scaling=-1), None, "scaling"), (dict(theta=0.0), None, "theta"),
    (dict(theta=float("nan")), None, "theta"), (dict(scaling=1, factor=0.0), None, "factor"),
    (dict(scaling=2, factor=2.0, dims=2), None, "ntk"), (dict(scaling=2, factor=1e300, theta=1e300), None, "out of range"), (dict(scaling=3, factor=2.0, length=0.0), None, "length"),
    (dict(scaling=3, factor=2.0, low=4.0, high=4.0), None, "low"), (dict(positions=None), None, "positions"),
    (dict(positions=P + 2), None, "positions"), (dict(positions=P + 4, positions_64=1), None, "positions"),
    ({}, dict(heads=-1), "heads"), ({}, dict(x=None), "null"), ({}, dict(out=None), "null"), ({}, dict(x=P + 1), "aligned"),
    ({}, dict(x_token=-1), "stride"), ({}, dict(out_head=-64), "stride"), ({}, dict(out=P, out_token=256), "strides"),
    ({}, dict(out_head=32), "stride"),
])
def test_rotary_refuses(lib, other, part, word):
    with pytest.raises(ValueError, match=word):
        _lib.check(lib.laya_op_rotary(ct.byref(rotary(part, **other)), None))
    with pytest.raises(ValueError, match="null"):
        _lib.check(lib.laya_op_rotary(None, None))


def attend(**other):
    fields = dict(sequences=2, heads=4, kv_heads=2, head_dim=64, dtype=2, q_tokens=10, k_tokens=20, max_queries=5, max_keys=10,
                  q=P, q_token=256, q_head=64, k=P, k_token=128, k_head=64, v=P, v_token=128, v_head=64, out=P, out_token=256, out_head=64,
                  starts=P, lengths=P, k_starts=P, k_lengths=P, scale=0.125, window_left=-1, window_right=-1)
    return _lib.Attend(**{**fields, **other})


@pytest.mark.parametrize("other,word", [
    (dict(sequences=-1), "shape"), (dict(sequences=65536), "shape"), (dict(q_tokens=-1), "shape"), (dict(k_tokens=-1), "shape"),
    (dict(q_tokens=2 ** 31 - 255), "tokens"), (dict(k_tokens=2 ** 31 - 1), "tokens"), (dict(max_queries=-1), "shape"), (dict(max_keys=-1), "shape"), (dict(heads=0), "heads"), (dict(kv_heads=0), "heads"),
    (dict(kv_heads=3), "heads"), (dict(heads=258), "128"), (dict(head_dim=0), "head"), (dict(head_dim=60), "multiple of 8"),
    (dict(head_dim=136), "128"), (dict(dtype=0), "dtype"), (dict(dtype=3), "dtype"), (dict(scale=float("inf")), "scale"),
    (dict(cap=-1.0), "cap"), (dict(cap=float("nan")), "cap"), (dict(window_left=-2), "window"), (dict(window_right=-5), "window"),
    (dict(slopes=P, distance_bias=P), "both"), (dict(distance_bias=P, reach=-1), "reach"), (dict(distance_bias=P, reach=2 ** 30), "reach"), (dict(documents=P), "documents"),
    (dict(k_documents=P), "documents"), (dict(k_starts=None), "k_lengths"), (dict(k_lengths=None), "k_starts"),
    (dict(starts=None), "null"), (dict(lengths=None), "null"), (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(out=None), "null"), (dict(q=P + 8), "16-byte"), (dict(k=P + 2), "16-byte"), (dict(v=P + 4), "16-byte"),
    (dict(out=P + 8), "16-byte"), (dict(q_token=260), "multiple of 8"), (dict(k_head=68), "multiple of 8"), (dict(v_token=0), "at least"),
    (dict(out_head=32), "at least"), (dict(k_token=-128), "at least"), (dict(k_token=1 << 40), "too large"),
])
def test_attend_refuses(lib, other, word):
    with pytest.raises(ValueError, match=word):
        _lib.check(lib.laya_op_attend(ct.byref(attend(**other)), None, None))
    with pytest.raises(ValueError, match="null"):
        _lib.check(lib.laya_op_attend(None, None, None))


@pytest.mark.parametrize("tokens,heads,token,head", [(4, 2, 64, 64), (10, 4, 128, 64), (10, 4, 64, 256), (2, 3, 128, 128), (3, 2, 128, 256), (5, 4, 256, 96), (5, 7, 200, 320),
                                                     (10 ** 6, 3, 64, 64 * 999999)])
def test_heads_that_overlap_are_not_written(lib, tokens, heads, token, head):
    if tokens < 100:  # by enumeration
        at = sorted(i * token + j * head for i in range(tokens) for j in range(heads))
        assert min(b - a for a, b in zip(at, at[1:])) < 64
    with pytest.raises(ValueError, match="overlap"):
        _lib.check(lib.laya_op_rotary(ct.byref(rotary(dict(out_token=token, out_head=head, heads=heads), tokens=tokens)), None))
    if token % 8 == 0 and head % 8 == 0:
        with pytest.raises(ValueError, match="overlap"):
            _lib.check(lib.laya_op_attend(ct.byref(attend(q_tokens=tokens, heads=heads, kv_heads=1, q_token=heads * 64, q_head=64, out_token=token, out_head=head)), None, None))
    for name in ("q", "k", "v"):  # what is read may overlap, but not lie within a head
        with pytest.raises(ValueError, match=f"{name}: strides .* at least"):
            _lib.check(lib.laya_op_attend(ct.byref(attend(**{name + "_head": 0})), None, None))


@pytest.mark.parametrize("name", ["starts", "lengths", "k_starts", "k_lengths", "prefix", "documents", "k_documents", "slopes", "distance_bias", "lse", "err"])
@pytest.mark.parametrize("off", [1, 2])
def test_attend_refuses_unaligned_vectors(lib, name, off):
    fields = dict(documents=P, k_documents=P) if "documents" in name else {}
    if name != "err":
        fields[name] = P + off
    with pytest.raises(ValueError, match=f"^{name} is not aligned"):
        _lib.check(lib.laya_op_attend(ct.byref(attend(**fields)), ct.c_void_p(P + off) if name == "err" else None, None))


def test_nothing_to_do_needs_no_buffers_and_no_device(lib):
    assert lib.laya_op_rotary(ct.byref(rotary(dict(x=None, out=None), tokens=0, positions=None)), None) == 0
    assert lib.laya_op_rotary(ct.byref(rotary(dict(x=None, out=None, heads=0), positions=None)), None) == 0
    none = dict(q=None, k=None, v=None, out=None, starts=None, lengths=None, k_starts=None, k_lengths=None)
    for other in (dict(sequences=0), dict(q_tokens=0), dict(max_queries=0)):
        assert lib.laya_op_attend(ct.byref(attend(**none, **other)), None, None) == 0


class Fake:
    """Stands for a CUDA tensor; counts nothing and holds nothing."""

    def __init__(self, shape, dtype="torch.bfloat16", size=2, device=0, stride=None, ptr=P):
        self.shape, self.dtype, self.size, self.device, self.ptr = tuple(shape), dtype, size, device, ptr
        self.strides = stride or tuple(int(np.prod(shape[k + 1:])) for k in range(len(shape)))

    def stride(self):
        return self.strides

    def element_size(self):
        return self.size

    def get_device(self):
        return self.device

    def data_ptr(self):
        return self.ptr


def ints(n, **other):
    return Fake((n,), "torch.int32", 4, **other)


X = Fake((6, 4, 64))


@pytest.mark.parametrize("call,error,word", [
    (dict(x=Fake((6, 256))), ValueError, "head_dim"), (dict(x=Fake((6, 4, 64), stride=(512, 128, 2))), ValueError, "contiguous"),
    (dict(x=Fake((6, 4, 64), "torch.int32", 4)), ValueError, "float"), (dict(x=Fake((6, 4, 64), device=-1)), ValueError, "CUDA"),
    (dict(out=Fake((6, 3, 64))), ValueError, "out must be"), (dict(out=Fake((6, 4, 64), "torch.float16")), ValueError, "type"),
    (dict(out=Fake((6, 4, 64), device=1)), ValueError, "device"), (dict(positions=ints(5)), ValueError, "positions"),
    (dict(positions=Fake((6,), "torch.float32", 4)), ValueError, "positions"), (dict(positions=ints(6, stride=(2,))), ValueError, "positions"),
    (dict(k=X), ValueError, "go together"), (dict(k=X, k_out=Fake((6, 2, 64))), ValueError, "k_out must be"),
    (dict(k=Fake((5, 4, 64)), k_out=X), ValueError, "k must be"), (dict(scaling="yes"), ValueError, "scaling"),
    (dict(scaling=1), ValueError, "scaling"), (dict(dims=2 ** 40), ValueError, "dims"), (dict(theta="x"), TypeError, "real number"),
    (dict(nothing=1), TypeError, "nothing"),
])
def test_python_rotary_refuses(call, error, word):
    with pytest.raises(error, match=word):
        attention.rotary(**{**dict(x=X, positions=ints(6), out=X), **call})


KV = Fake((9, 2, 64))


@pytest.mark.parametrize("call,error,word", [
    (dict(q=Fake((6, 4, 64), stride=(512, 128, 2))), ValueError, "contiguous"), (dict(k=Fake((9, 2, 32))), ValueError, "k must be"),
    (dict(v=Fake((8, 2, 64))), ValueError, "v must be"), (dict(v=Fake((9, 2, 64), "torch.float16")), ValueError, "type"),
    (dict(out=Fake((6, 2, 64))), ValueError, "out must be"), (dict(k=Fake((9, 2, 64), device=1)), ValueError, "device"),
    (dict(starts=Fake((2, 1), "torch.int32", 4)), ValueError, "starts"), (dict(starts=Fake((2,), "torch.int64", 8)), ValueError, "starts"),
    (dict(lengths=ints(3)), ValueError, "lengths"), (dict(lengths=None), ValueError, "lengths"), (dict(k_starts=ints(2)), ValueError, "go together"),
    (dict(k_starts=ints(2), k_lengths=ints(1)), ValueError, "k_lengths"), (dict(prefix=ints(1)), ValueError, "prefix"),
    (dict(documents=ints(6)), ValueError, "k_documents"), (dict(documents=ints(5), k_documents=ints(9)), ValueError, "documents"),
    (dict(documents=ints(6), k_documents=ints(6)), ValueError, "k_documents"), (dict(slopes=ints(4)), ValueError, "slopes"),
    (dict(slopes=Fake((2,), "torch.float32", 4)), ValueError, "slopes"), (dict(distance_bias=Fake((4, 4), "torch.float32", 4)), ValueError, "reach"),
    (dict(distance_bias=Fake((2, 5), "torch.float32", 4)), ValueError, "reach"), (dict(lse=Fake((6, 2), "torch.float32", 4)), ValueError, "lse"),
    (dict(err=Fake((1,), "torch.int64", 8)), ValueError, "err"), (dict(window=(1, 2, 3)), ValueError, "window"),
    (dict(window=1.5), ValueError, "window"), (dict(cap="x"), TypeError, "real number"), (dict(max_queries=2 ** 40), ValueError, "max_queries"),
])
def test_python_attend_refuses(call, error, word):
    with pytest.raises(error, match=word):
        attention.attend(**{**dict(q=X, k=KV, v=KV, out=X, starts=ints(2), lengths=ints(2)), **call})
