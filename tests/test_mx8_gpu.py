"""The MX8 operators on the GPU against their definitions in 64 bits.

Quantising and reading back are exact operations and are compared bit for bit.  The norm and the
product compute in fp32; their tolerances are bounds on that arithmetic (see `norm_slack` and
`product_slack`) plus the one rounding of the output.
"""
import ctypes as ct
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from laya_cuda import _lib, mx8  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Half a unit in the last place of a rounded output, relative.
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")


# -------------------------------------------------------------------------------- the format in 64 bits

def e4m3_table():
    out = np.empty(256)
    for b in range(256):
        sign, power, fraction = -1.0 if b & 128 else 1.0, (b >> 3) & 15, b & 7
        v = (1 + fraction / 8) * 2.0 ** (power - 7) if power else fraction / 8 * 2.0 ** -6
        out[b] = math.nan if (b & 127) == 127 else sign * v
    return out


TABLE = e4m3_table()


def scale_index(rows, cols):
    """Byte index of each (row, block)."""
    r, b = np.arange(rows)[:, None], np.arange(-(-cols // 32))[None, :]
    return (r // 128 * -(-cols // 128) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4


def decode(m):
    """A Matrix in float64, [rows][cols], and its scale exponents [rows][blocks] (255: NaN)."""
    q = m.values.cpu().numpy()[:, : m.cols]
    byte = m.scales.cpu().numpy()[scale_index(m.rows, m.cols)].astype(np.int64)
    scale = np.where(byte == 255, math.nan, np.ldexp(1.0, byte - 127))
    return TABLE[q] * np.repeat(scale, 32, axis=1)[:, : m.cols], byte


def blocks(v):
    rows, cols = v.shape
    out = np.zeros((rows, -(-cols // 32) * 32))
    out[:, :cols] = v
    return out.reshape(rows, -1, 32)


def define(v):
    """The definition: E4M3 codes and scale bytes of float64 values."""
    b = blocks(v)
    bad = ~np.isfinite(b).all(-1)
    a = np.abs(np.where(np.isfinite(b), b, 0)).max(-1)
    mantissa, power = np.frexp(a)
    e = np.where(a > 0, power - 9 + (mantissa > 0.875), -127)
    e = np.maximum(e, -127)
    x = np.where(bad[..., None], 0, b) / np.ldexp(1.0, e)[..., None]
    # Nearest E4M3 magnitude, ties to the even code (codes 0..126 ascend).
    mags = TABLE[:127]
    hi = np.clip(np.searchsorted(mags, np.abs(x)), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = np.abs(x) - mags[lo], mags[hi] - np.abs(x)
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(x), code + 128, code)
    code = np.where(bad[..., None], 127, code)
    return code.reshape(v.shape[0], -1)[:, : v.shape[1]].astype(np.uint8), np.where(bad, 255, e + 127)


def matrix(v):
    """A Matrix that holds float64/float32 values `v` (numpy), and what it stands for."""
    rows, cols = v.shape
    code, byte = define(v.astype(np.float64))
    room = (cols + 15) // 16 * 16
    q = np.zeros((rows, room), np.uint8)
    q[:, :cols] = code
    s = np.full(mx8.scale_bytes(rows, cols), 255, np.uint8)  # unwritten rows may hold anything
    idx = scale_index(rows, -(-cols // 128) * 128)
    s[idx] = 0
    s[scale_index(rows, cols)] = byte
    m = mx8.Matrix(torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), rows, cols)
    return m, decode(m)[0]


def fresh(rows, cols):
    m = mx8.Matrix.empty(torch.empty(0, device="cuda"), rows, cols)
    m.values.fill_(0xA5)
    m.scales.fill_(0xA5)
    return m


def strided(rows, cols, dtype, pad=0, offset=0, fill=None):
    """[rows][cols] view with row stride cols + pad, starting `offset` elements into its buffer."""
    store = torch.full((rows * (cols + pad) + offset + 8,), 7.0, dtype=dtype, device="cuda")
    view = store[offset: offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    if fill is not None:
        view.copy_(torch.from_numpy(fill))
    return view, store


def untouched(view, store, pad, offset):
    """Every element of the buffer outside the view still holds 7."""
    rest = store.clone()
    rows, cols = view.shape
    rest[offset: offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] = 7.0
    return bool((rest == 7.0).all())


def activations(rng, rows, cols):
    return (rng.normal(0, 1, (rows, cols)) * np.exp(0.8 * rng.normal(0, 1, cols))).astype(np.float32)


SHAPES = [(1, 1), (1, 31), (3, 32), (5, 33), (1, 768), (129, 100), (257, 128), (33, 1000), (1, 5000), (300, 264)]


# -------------------------------------------------------------------------------- quantize, dequantize

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1), (8, 8)])
def test_quantize_is_the_definition_bit_for_bit(dtype, rows, cols, pad, offset):
    rng = np.random.default_rng(rows * 1000 + cols)
    v = activations(rng, rows, cols) * np.ldexp(1.0, rng.integers(-12, 5, (rows, 1))).astype(np.float32)
    v[rng.random((rows, cols)) < 0.05] = 0
    if cols >= 64:
        v[0, :32] = 0  # a block of zeros
    x, _ = strided(rows, cols, TYPES[dtype], pad, offset, v)
    out = fresh(rows, cols)
    mx8.quantize(x, out)
    code, byte = define(x.double().cpu().numpy())
    got = out.values.cpu().numpy()
    np.testing.assert_array_equal(got[:, :cols], code)
    assert not got[:, cols:].any()
    np.testing.assert_array_equal(out.scales.cpu().numpy()[scale_index(rows, cols)], byte)
    whole = out.scales.cpu().numpy()[scale_index(rows, -(-cols // 128) * 128)]
    assert not whole[:, -(-cols // 32):].any()


def test_quantize_at_the_edges_of_the_range():
    """Largest magnitudes around 1.75 x 2^p, ties, subnormals, the extremes of fp32 and signed zeros."""
    up = np.nextafter(np.float32(1.75), np.float32(2))
    rows = [[1.75], [up], [np.float32(2.0 ** -126)], [np.float32(1e-45)], [np.float32(3.4028235e38)], [-0.0],
            [448.0, 17.0, 18.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10], [np.float32(1.75 * 2.0 ** -119)], [np.float32(2.0 ** -119)]]
    v = np.zeros((len(rows), 32), np.float32)
    for i, r in enumerate(rows):
        v[i, :len(r)] = r
    out = fresh(*v.shape)
    mx8.quantize(torch.from_numpy(v).cuda(), out)
    code, byte = define(v.astype(np.float64))
    np.testing.assert_array_equal(out.values.cpu().numpy(), code)
    np.testing.assert_array_equal(out.scales.cpu().numpy()[scale_index(*v.shape)], byte)
    assert byte[0, 0] == 119 and byte[1, 0] == 120


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_non_finite_blocks_read_back_as_nan_and_no_other(bad):
    v = np.ones((4, 96), np.float32)
    v[2, 40] = bad
    out, back = fresh(4, 96), torch.empty(4, 96, device="cuda")
    mx8.quantize(torch.from_numpy(v).cuda(), out)
    mx8.dequantize(out, back)
    want = v.copy()
    want[2, 32:64] = math.nan
    np.testing.assert_array_equal(back.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1)])
def test_dequantize_is_exact(dtype, rows, cols, pad, offset):
    rng = np.random.default_rng(rows * 1000 + cols + 1)
    m, v = matrix(activations(rng, rows, cols))
    out, store = strided(rows, cols, TYPES[dtype], pad, offset)
    mx8.dequantize(m, out)
    want = torch.from_numpy(v).to(TYPES[dtype])
    assert torch.equal(out.cpu(), want)
    assert untouched(out, store, pad, offset)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols,pad", [(67, 199, 0), (67, 200, 0), (67, 201, 2), (40, 217, 0), (40, 233, 7), (9, 511, 0), (9, 512, 1), (9, 513, 0),
                                           (5, 1025, 3), (3, 4095, 0)])
def test_dequantize_into_every_alignment(dtype, rows, cols, pad):
    """Each place in a 32-byte sector at which a row can start; what lies around the rows stays."""
    rng = np.random.default_rng(rows * 1000 + cols + 2)
    m, v = matrix(activations(rng, rows, cols))
    want = torch.from_numpy(v).to(TYPES[dtype])
    for offset in range(16):
        out, store = strided(rows, cols, TYPES[dtype], pad, offset)
        mx8.dequantize(m, out)
        assert torch.equal(out.cpu(), want), offset
        assert untouched(out, store, pad, offset), offset


def test_dequantize_every_code_and_scale():
    """Each E4M3 code under each scale byte (fp32 output; overflow to infinity as the rounding gives)."""
    q = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    m = mx8.Matrix(q.cuda(), torch.zeros(mx8.scale_bytes(256, 256), dtype=torch.uint8, device="cuda"), 256, 256)
    byte = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 8, axis=1)
    s = m.scales.cpu().numpy()
    s[scale_index(256, 256)] = byte
    m.scales.copy_(torch.from_numpy(s))
    out = torch.empty(256, 256, device="cuda")
    mx8.dequantize(m, out)
    with np.errstate(over="ignore"):
        want = decode(m)[0].astype(np.float32)
    np.testing.assert_array_equal(out.cpu().numpy(), want)


# -------------------------------------------------------------------------------- rms_norm

def norm_slack(cols):
    """Relative error of y: the sum of squares is a tree over at most cols / 32 + 32 serial additions
    and products, halved by the root; then four roundings."""
    return (cols / 32 + 32) * 2.0 ** -24 / 2 + 5 * 2.0 ** -24


def check_mx8(out, y, slack):
    """`out` holds y (float64) to within `slack` (absolute, per element) and E4M3's rounding."""
    got, byte = decode(out)
    a = np.abs(blocks(y)).max(-1)
    da = blocks(np.broadcast_to(slack, y.shape)).max(-1)
    lo, hi = define(np.maximum(a - da, 0).reshape(-1, 1))[1], define((a + da).reshape(-1, 1))[1]
    assert ((byte >= lo.reshape(byte.shape)) & (byte <= hi.reshape(byte.shape))).all()
    scale = np.repeat(np.ldexp(1.0, byte - 127), 32, axis=1)[:, : y.shape[1]]
    power = np.floor(np.log2(np.maximum(np.abs(y) / scale, 2.0 ** -6)))
    # Half a step: 2^(power - 4), one binade up where the slack may cross it.
    half = scale * np.ldexp(1.0, power.astype(np.int64) - 4)
    off = np.abs(got - y)
    tol = half * (1 + 1e-12) + 2 * slack
    assert (off <= tol).all(), float((off / tol).max())
    q = out.values.cpu().numpy()
    assert not q[:, out.cols: (out.cols + 15) // 16 * 16].any()


NORM_SHAPES = [(1, 1), (2, 31), (7, 33), (1, 768), (130, 256), (300, 100), (77, 128), (50, 250), (3, 12001), (33, 1000), (3, 2048), (2, 4100), (5, 8192), (1, 16384), (2, 40000)]


@pytest.mark.parametrize("dtype,rdtype", [("bf16", "f32"), ("f16", "f16"), ("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (5, 1)])
def test_rms_norm(dtype, rdtype, rows, cols, pad, offset):
    rng = np.random.default_rng(rows * 31 + cols)
    x, _ = strided(rows, cols, TYPES[dtype], pad, offset, activations(rng, rows, cols))
    r, _ = strided(rows, cols, TYPES[rdtype], pad, offset, rng.normal(0, 1, (rows, cols)).astype(np.float32))
    w = torch.from_numpy((1 + 0.2 * rng.normal(0, 1, cols)).astype(np.float32)).cuda()
    total, store = strided(rows, cols, TYPES[rdtype], pad, offset)
    out = fresh(rows, cols)
    mx8.rms_norm(x, w, out, residual=r, sum_out=total, eps=1e-5)
    h = x.double().cpu().numpy() + r.double().cpu().numpy()
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-5) * w.double().cpu().numpy()
    off = np.abs(total.double().cpu().numpy() - h)
    assert (off <= (HALF_ULP[rdtype] + 2.0 ** -23) * np.abs(h) + TINY[rdtype]).all()
    assert untouched(total, store, pad, offset)
    # h itself is rounded to fp32 once before it is squared and scaled.
    check_mx8(out, y, norm_slack(cols) * np.abs(y))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("cols", [16385, 16400, 20001])
def test_rms_norm_sum_of_long_rows_at_every_alignment(dtype, cols):
    """The sum is one fp32 addition and one rounding, whatever the place in a sector at which a row starts; here
    also over the residual itself."""
    rng = np.random.default_rng(cols)
    x = torch.from_numpy(activations(rng, 3, cols)).to(TYPES[dtype]).cuda()
    r = rng.normal(0, 1, (3, cols)).astype(np.float32)
    want = (x.float() + torch.from_numpy(r).to(TYPES[dtype]).cuda().float()).to(TYPES[dtype])
    w = torch.ones(cols, device="cuda")
    first = None
    for offset in range(16):
        stream, store = strided(3, cols, TYPES[dtype], 1, offset, r)
        out = fresh(3, cols)
        mx8.rms_norm(x, w, out, residual=stream, sum_out=stream, eps=1e-5)
        assert torch.equal(stream, want), offset
        assert untouched(stream, store, 1, offset), offset
        first = out if first is None else first
        assert torch.equal(out.values, first.values) and torch.equal(out.scales, first.scales), offset


def test_rms_norm_without_residual_and_in_place():
    rng = np.random.default_rng(5)
    rows, cols = 9, 520
    v = activations(rng, rows, cols)
    x, w = torch.from_numpy(v).cuda(), torch.ones(cols, device="cuda")
    out = fresh(rows, cols)
    mx8.rms_norm(x, w, out)
    h = v.astype(np.float64)
    check_mx8(out, h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-6), norm_slack(cols) * np.abs(h) * 2)
    r = torch.from_numpy(rng.normal(0, 1, (rows, cols)).astype(np.float32)).cuda()
    keep, one, two = r.clone(), fresh(rows, cols), torch.empty_like(r)
    mx8.rms_norm(x, w, one, residual=r, sum_out=two)
    mx8.rms_norm(x, w, out, residual=r, sum_out=r)
    assert torch.equal(r, two) and torch.equal(out.values, one.values) and not torch.equal(r, keep)


def test_rms_norm_of_zero_rows_is_zero_and_non_finite_rows_are_nan():
    x = torch.ones(5, 300, device="cuda")
    x[1] = 0
    x[3, 7] = math.inf
    x[4, 299] = math.nan
    out, back = fresh(5, 300), torch.empty(5, 300, device="cuda")
    mx8.rms_norm(x, torch.ones(300, device="cuda"), out, eps=0.0)
    mx8.dequantize(out, back)
    got = back.cpu()
    assert torch.equal(got[0], torch.ones(300)) and torch.equal(got[2], torch.ones(300))
    assert torch.isnan(got[4]).all()
    # 0 * rsqrt(0) is NaN without eps; with eps it is 0.
    assert torch.isnan(got[1]).all()
    mx8.rms_norm(x, torch.ones(300, device="cuda"), out)
    mx8.dequantize(out, back)
    assert not back[1].any()
    # inf / inf is NaN; the finite values of that row are over infinity, 0, outside the NaN's block.
    assert torch.isnan(back[3, :32]).all() and not back[3, 32:].any()


# -------------------------------------------------------------------------------- linear

def act64(v, name):
    if name == "relu":
        return np.maximum(v, 0)
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(torch.from_numpy(v / math.sqrt(2))).numpy())
    if name == "silu":
        return v / (1 + np.exp(-v))
    return v


def product_slack(x, w):
    """Error of the fp32 sums: K / 32 accumulation steps, each off by at most 2^-22 (a unit in the last place of
    a truncated fp32 sum and of its aligned terms) of the largest partial sum, which for these inputs stays
    under four times the root of the sum of the squared products."""
    k = x.shape[1]
    return (k / 32 + 1) * 2.0 ** -20 * np.sqrt((x * x) @ (w * w).T)


def reference(x, w, gate, bias, gate_bias, act, residual):
    """The result in float64 and its slack before the output's rounding."""
    u, du = x @ w.T, product_slack(x, w)
    if bias is not None:
        u, du = u + bias, du + 2.0 ** -23 * np.abs(u + bias)
    if gate is not None:
        g, dg = x @ gate.T, product_slack(x, gate)
        if gate_bias is not None:
            g, dg = g + gate_bias, dg + 2.0 ** -23 * np.abs(g + gate_bias)
        a = act64(g, act)
        # Activations have slopes up to 1.13 and are themselves within 1e-6 (absolute, or relative where larger).
        da = 1.13 * dg + 1e-6 * (1 + np.abs(a))
        y, dy = a * u, np.abs(u) * da + np.abs(a) * du + da * du
    else:
        y = act64(u, act)
        dy = 1.13 * du + (0 if act == "none" else 1e-6 * (1 + np.abs(y)))
    if residual is not None:
        y, dy = y + residual, dy + 2.0 ** -23 * np.abs(y + residual)
    return y, dy + 2.0 ** -22 * np.abs(y)


def run_linear(rows, cols, n, out_type, act="none", gated=False, bias=False, residual=None, seed=0, pad=0, offset=0):
    rng = np.random.default_rng(seed + rows * 7 + cols * 3 + n)
    x, xd = matrix(activations(rng, rows, cols))
    w, wd = matrix((rng.normal(0, 1, (n, cols)) / math.sqrt(cols)).astype(np.float32))
    g, gd = matrix((rng.normal(0, 1, (n, cols)) / math.sqrt(cols)).astype(np.float32)) if gated else (None, None)
    vec = lambda on: torch.from_numpy((0.1 * rng.normal(0, 1, n)).astype(np.float32)).cuda() if on else None  # noqa: E731
    b, gb = vec(bias), vec(bias and gated)
    r = None
    if residual:
        r, _ = strided(rows, n, TYPES[residual], pad, offset, rng.normal(0, 1, (rows, n)).astype(np.float32))
    to64 = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    y, dy = reference(xd, wd, gd, to64(b), to64(gb), act, to64(r))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    if out_type == "mx8":
        out, store = fresh(rows, n), None
    else:
        out, store = strided(rows, n, TYPES[out_type], pad, offset)
    mx8.linear(x, w, out, bias=b, gate=g, gate_bias=gb, activation=act, residual=r, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    if out_type == "mx8":
        check_mx8(out, y, dy)
    else:
        off = np.abs(out.double().cpu().numpy() - y)
        tol = dy + HALF_ULP[out_type] * (np.abs(y) + dy) + TINY[out_type]
        assert (off <= tol).all(), float((off / tol).max())
        assert untouched(out, store, pad, offset)


LINEAR_SHAPES = [(1, 1, 1), (1, 32, 8), (1, 768, 768), (2, 33, 31), (7, 128, 129), (16, 1000, 257), (17, 160, 64), (31, 31, 300),
                 (33, 512, 200), (64, 2048, 384), (65, 256, 130), (100, 777, 513), (128, 128, 128), (129, 96, 257),
                 (200, 1024, 640), (257, 4096, 96), (300, 260, 1000), (513, 640, 300)]


@pytest.mark.parametrize("rows,cols,n", LINEAR_SHAPES)
@pytest.mark.parametrize("out_type", ["bf16", "f32", "mx8"])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_shapes(rows, cols, n, out_type, gated):
    run_linear(rows, cols, n, out_type, act="silu" if gated else "none", gated=gated)


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("out_type,residual", [("f16", None), ("bf16", "f32"), ("f32", "bf16"), ("mx8", "f16")])
def test_linear_epilogues(rows, act, gated, out_type, residual):
    run_linear(rows, 320, 264, out_type, act=act, gated=gated, bias=True, residual=residual, seed=1)


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("pad,offset", [(1, 1), (4, 0), (3, 2), (8, 8)])
@pytest.mark.parametrize("out_type", ["f16", "f32"])
def test_linear_strides_and_alignment(rows, pad, offset, out_type):
    run_linear(rows, 200, 133, out_type, bias=True, residual="bf16", seed=2, pad=pad, offset=offset)


def decode_gpu(m):
    """decode() on the GPU, for the larger cases: float64 values."""
    q = torch.from_numpy(TABLE).cuda()[m.values[:, : m.cols].long()]
    byte = m.scales[torch.from_numpy(scale_index(m.rows, m.cols)).cuda()].double()
    return q * torch.exp2(byte - 127).repeat_interleave(32, dim=1)[:, : m.cols]


LARGE = [  # rows, cols, features: 256 x 128 tiles; 256 x 256 tiles; gated tiles
    (2500, 160, 500, False), (2560, 128, 512, False), (2309, 70, 600, False),
    (1024, 4096, 4096, False), (1030, 4100, 4130, False), (4096, 1024, 3584, False),
    (1500, 300, 700, True), (2100, 640, 1056, True)]


@pytest.mark.parametrize("rows,cols,n,gated", LARGE)
@pytest.mark.parametrize("out_type,act,bias,residual,pad,offset", [
    ("bf16", "none", False, None, 0, 0), ("f16", "silu", True, "bf16", 0, 0), ("f32", "none", True, "f32", 0, 0),
    ("mx8", "relu", False, "f16", 0, 0), ("mx8", "gelu", True, None, 0, 0), ("bf16", "none", False, "f16", 3, 1),
    ("f32", "gelu", False, "f32", 1, 1), ("f16", "none", False, "f32", 32, 16)])
def test_linear_large(rows, cols, n, gated, out_type, act, bias, residual, pad, offset):
    """Results too large for the few-row kernel, over its tile forms, against float64 on the GPU; the operands'
    float64 values are read back from what `quantize` wrote."""
    g = torch.Generator(device="cuda").manual_seed(rows + cols + n)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    x, w, gate = fresh(rows, cols), fresh(n, cols), fresh(n, cols) if gated else None
    mx8.quantize(rand(rows, cols) * torch.exp(0.8 * rand(cols)), x)
    for m in (w, gate) if gated else (w,):
        mx8.quantize(rand(n, cols) / math.sqrt(cols), m)
    b, gb = 0.1 * rand(n) if bias else None, 0.1 * rand(n) if bias and gated else None
    r = None
    if residual:
        r, _ = strided(rows, n, TYPES[residual], pad, offset)
        r.copy_(rand(rows, n))
    xd, to64 = decode_gpu(x), lambda t: None if t is None else t.double()

    def product(m, add):
        md = decode_gpu(m)
        v, d = xd @ md.T, (cols / 32 + 1) * 2.0 ** -20 * ((xd * xd) @ (md * md).T).sqrt()
        return (v, d) if add is None else (v + add, d + 2.0 ** -23 * (v + add).abs())

    def apply(v):
        f = {"relu": lambda t: t.clamp(min=0), "gelu": lambda t: 0.5 * t * torch.erfc(-t / math.sqrt(2)),
             "silu": lambda t: t * torch.sigmoid(t)}
        return f[act](v) if act in f else v

    # The slack of `reference`, on the GPU.
    u, du = product(w, to64(b))
    if gated:
        p, dp = product(gate, to64(gb))
        a = apply(p)
        da = 1.13 * dp + 1e-6 * (1 + a.abs())
        y, dy = a * u, u.abs() * da + a.abs() * du + da * du
    else:
        y = apply(u)
        dy = 1.13 * du + (0 if act == "none" else 1e-6 * (1 + y.abs()))
    if r is not None:
        y, dy = y + r.double(), dy + 2.0 ** -23 * (y + r.double()).abs()
    dy = dy + 2.0 ** -22 * y.abs()

    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, store = (fresh(rows, n), None) if out_type == "mx8" else strided(rows, n, TYPES[out_type], pad, offset)
    mx8.linear(x, w, out, bias=b, gate=gate, gate_bias=gb, activation=act, residual=r, err=err)
    assert int(err.item()) == 0
    if out_type == "mx8":
        check_mx8(out, y.cpu().numpy(), dy.cpu().numpy())
    else:
        off, tol = (out.double() - y).abs(), dy + HALF_ULP[out_type] * (y.abs() + dy) + TINY[out_type]
        assert bool((off <= tol).all()), float((off / tol).max())
        assert untouched(out, store, pad, offset)
    if r is not None and out_type == residual:
        mx8.linear(x, w, r, bias=b, gate=gate, gate_bias=gb, activation=act, residual=r)
        assert torch.equal(r, out)


@pytest.mark.parametrize("rows,n", [(3, 256), (260, 255), (2600, 512), (2600, 511), (6000, 129)])
def test_linear_adds_into_the_residual_in_place(rows, n):
    rng = np.random.default_rng(8)
    x, _ = matrix(activations(rng, rows, 192))
    w, _ = matrix(rng.normal(0, 0.1, (n, 192)).astype(np.float32))
    r = torch.from_numpy(rng.normal(0, 1, (rows, n)).astype(np.float32)).cuda()
    want = torch.empty_like(r)
    mx8.linear(x, w, want, residual=r)
    mx8.linear(x, w, r, residual=r)
    assert torch.equal(r, want)


@pytest.mark.parametrize("rows", [5, 150, 400, 3400])
def test_linear_keeps_non_finite_values_to_their_rows(rows):
    """A NaN block of x makes its row NaN, one of w its column; nothing else changes.  The scales of rows past
    the last hold NaN bytes (see `matrix`) and reach no result."""
    rng = np.random.default_rng(9)
    xv, wv = activations(rng, rows, 256), rng.normal(0, 0.1, (300, 256)).astype(np.float32)
    plain = torch.empty(rows, 300, device="cuda")
    mx8.linear(matrix(xv)[0], matrix(wv)[0], plain)
    assert torch.isfinite(plain).all()
    xv[2, 70], wv[291, 3] = math.inf, math.nan
    out = torch.empty(rows, 300, device="cuda")
    mx8.linear(matrix(xv)[0], matrix(wv)[0], out)
    want = plain.clone()
    want[2], want[:, 291] = math.nan, math.nan
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(want))


@pytest.mark.parametrize("rows,cols,n", [(4, 2048, 512), (90, 1024, 512), (700, 512, 768), (2600, 512, 768)])
def test_linear_gives_the_same_bits_each_time_and_a_row_does_not_depend_on_the_others(rows, cols, n):
    rng = np.random.default_rng(10)
    xv = activations(rng, rows, cols)
    w, _ = matrix(rng.normal(0, 0.1, (n, cols)).astype(np.float32))
    x, _ = matrix(xv)
    one, two, other = (torch.empty(rows, n, device="cuda") for _ in range(3))
    mx8.linear(x, w, one)
    xv[1:] *= -3
    mx8.linear(matrix(xv)[0], w, other)
    mx8.linear(x, w, two)
    assert torch.equal(one, two) and torch.equal(one[0], other[0])


def test_one_layer_on_another_stream():
    """norm -> gated product in MX8 -> product onto the residual, on a side stream."""
    rng = np.random.default_rng(11)
    rows, d, f = 70, 256, 352
    x = torch.from_numpy(activations(rng, rows, d)).cuda().bfloat16()
    r = torch.from_numpy(rng.normal(0, 1, (rows, d)).astype(np.float32)).cuda()
    weight = torch.ones(d, device="cuda")
    (up, _), (gate, _), (down, downd) = (matrix(rng.normal(0, 0.08, s).astype(np.float32)) for s in ((f, d), (f, d), (d, f)))
    n8, a8, y = fresh(rows, d), fresh(rows, f), torch.empty(rows, d, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    s = side.cuda_stream
    mx8.rms_norm(x, weight, n8, residual=r, sum_out=r, stream=s)
    mx8.linear(n8, up, a8, gate=gate, activation="silu", stream=s)
    mx8.linear(a8, down, y, residual=r, stream=s)
    side.synchronize()
    a = decode(a8)[0]
    want, slack = reference(a, downd, None, None, None, "none", r.double().cpu().numpy())
    assert (np.abs(y.double().cpu().numpy() - want) <= slack + 2.0 ** -23 * np.abs(want)).all()


@pytest.mark.parametrize("rows", [1, 40, 300, 10000])
def test_captured_in_a_graph(rows):
    """The calls can be captured and replayed on new inputs, and give the bits of plain calls."""
    rng = np.random.default_rng(12)
    d, f = 192, 256
    (up, _), (down, _) = (matrix(rng.normal(0, 0.1, s).astype(np.float32)) for s in ((f, d), (d, f)))
    x, r = (torch.from_numpy(activations(rng, rows, d)).cuda() for _ in range(2))
    weight = torch.ones(d, device="cuda")
    n8, a8 = fresh(rows, d), fresh(rows, f)
    y, back = torch.empty(rows, d, device="cuda"), torch.empty(rows, f, device="cuda")

    def layer(s):
        mx8.rms_norm(x, weight, n8, residual=r, stream=s)
        mx8.linear(n8, up, a8, activation="gelu", stream=s)
        mx8.dequantize(a8, back, stream=s)
        mx8.quantize(back, a8, stream=s)
        mx8.linear(a8, down, y, residual=r, stream=s)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer(side.cuda_stream)
    x.mul_(0.5)
    graph.replay()
    got = y.clone()
    layer(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(got, y) and torch.isfinite(y).all()


def test_offsets_past_32_bits():
    """Rows 2^31 bytes and more apart: values, tensors and results."""
    rng = np.random.default_rng(13)
    rows, cols, n, apart = 3, 96, 64, 2 ** 30 + 64
    v, w = activations(rng, rows, cols), matrix(rng.normal(0, 0.1, (n, cols)).astype(np.float32))[0]
    near = torch.from_numpy(v).cuda().bfloat16()
    store = torch.empty((rows - 1) * apart + cols, dtype=torch.bfloat16, device="cuda")
    far = store.as_strided((rows, cols), (apart, 1))
    far.copy_(near)
    byte = torch.zeros((rows - 1) * (2 ** 31 + 64) + 96, dtype=torch.uint8, device="cuda")
    far8 = mx8.Matrix(byte.as_strided((rows, cols), (2 ** 31 + 64, 1)), torch.zeros(512, dtype=torch.uint8, device="cuda"), rows, cols)
    near8 = fresh(rows, cols)
    weight = torch.ones(cols, device="cuda")
    for to8, x in ((far8, far), (near8, near)):
        mx8.rms_norm(x, weight, to8, residual=x, sum_out=x)
        mx8.quantize(x, to8)
    assert torch.equal(far, near) and torch.equal(far8.values, near8.values)
    got, want = store.as_strided((rows, n), (apart, 1)), torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    mx8.dequantize(far8, far)
    mx8.dequantize(near8, near)
    assert torch.equal(far, near)
    mx8.linear(far8, w, got, residual=far[:, :n].clone())
    mx8.linear(near8, w, want, residual=near[:, :n].clone())
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows,cols,n,gated", [(3, 65536, 256, False), (40, 65536, 300, True), (300, 65536, 520, False), (3000, 32768, 520, False), (2600, 16384, 512, True)])
def test_a_wait_that_runs_out_is_reported_and_leaves_the_device_usable(rows, cols, n, gated):
    """Valid calls, deep enough that the epilogue waits for many microseconds, whose waits are limited to a nanosecond: the
    kernel unwinds and sets `err`; the next call, with the default limit, gives the bits of a call before it."""
    lib = _lib.load()
    generator = torch.Generator(device="cuda").manual_seed(14)
    x, w = fresh(rows, cols), fresh(n, cols)
    for m in (x, w):
        mx8.quantize(torch.randn(m.rows, cols, generator=generator, device="cuda"), m)
    gate = w if gated else None
    want, got = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    mx8.linear(x, w, want, gate=gate, activation="silu", err=err)
    assert int(err.item()) == 0
    try:
        assert lib.laya_set_launch_options(1, 1) == 0
        mx8.linear(x, w, got, gate=gate, activation="silu", err=err)
        torch.cuda.synchronize()
    finally:
        assert lib.laya_set_launch_options(1, 0) == 0
    assert 1 <= int(err.item()) <= 3
    err.zero_()
    mx8.linear(x, w, got, gate=gate, activation="silu", err=err)
    assert int(err.item()) == 0 and torch.equal(got, want)


def test_no_rows_is_no_work():
    w, _ = matrix(np.ones((8, 32), np.float32))
    x = mx8.Matrix.empty(w.values, 0, 32)
    mx8.linear(x, w, torch.empty(0, 8, device="cuda"))
    mx8.quantize(torch.empty(0, 32, device="cuda"), x)
    mx8.dequantize(x, torch.empty(0, 32, device="cuda"))
    mx8.rms_norm(torch.empty(0, 32, device="cuda"), torch.ones(32, device="cuda"), x)
    torch.cuda.synchronize()


def test_refusals():
    w, _ = matrix(np.ones((8, 32), np.float32))
    x, _ = matrix(np.ones((3, 32), np.float32))
    other, _ = matrix(np.ones((3, 64), np.float32))
    good = torch.empty(3, 8, device="cuda")
    for bad in (lambda: mx8.linear(other, w, good),
                lambda: mx8.linear(x, w, torch.empty(3, 9, device="cuda")),
                lambda: mx8.linear(x, w, good.double()),
                lambda: mx8.linear(x, w, torch.empty(8, 3, device="cuda").T),
                lambda: mx8.linear(x, w, good, activation="tanh"),
                lambda: mx8.linear(x, w, good, gate=other),
                lambda: mx8.linear(x, w, good, gate_bias=torch.zeros(8, device="cuda")),
                lambda: mx8.linear(x, w, good, bias=torch.zeros(8, device="cuda").half()),
                lambda: mx8.linear(x, w, good, bias=torch.zeros(9, device="cuda")[1:]),
                lambda: mx8.linear(x, w, good, residual=torch.zeros(1, 8, device="cuda").expand(3, 8)),
                lambda: mx8.linear(x, w, good.cpu()),
                lambda: mx8.quantize(torch.ones(3, 31, device="cuda"), x),
                lambda: mx8.quantize(torch.ones(3, 32, device="cuda", dtype=torch.int32), x),
                lambda: mx8.rms_norm(torch.ones(3, 32, device="cuda"), torch.ones(31, device="cuda"), x),
                lambda: mx8.rms_norm(torch.ones(3, 32, device="cuda"), torch.ones(32, device="cuda"), x, eps=-1.0),
                lambda: mx8.rms_norm(torch.ones(3, 32, device="cuda"), torch.ones(32, device="cuda"), x,
                                     residual=torch.ones(3, 32, device="cuda"),
                                     sum_out=torch.ones(3, 32, device="cuda").half()),
                lambda: mx8.Matrix(x.values[:, 1:], x.scales, 3, 31),
                lambda: mx8.Matrix(x.values, x.scales[:511], 3, 32),
                lambda: mx8.Matrix.empty(good, 3, 0)):
        with pytest.raises(ValueError):
            bad()
    # A matrix whose rows are not 16-byte aligned is refused when it is used.
    shifted = torch.zeros(3 * 48 + 1, dtype=torch.uint8, device="cuda")[1:].view(3, 48)
    with pytest.raises(ValueError, match="aligned"):
        mx8.linear(mx8.Matrix(shifted, x.scales, 3, 32), w, good)


def test_the_feed_forward_example(capsys):
    """The example runs, and its block is the operators one after the other, bit for bit."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parents[1] / "examples" / "mx8_feed_forward.py"
    spec = importlib.util.spec_from_file_location("mx8_feed_forward", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    seen = dict(example.main(384, 1000))
    assert set(seen) == {1, 512, 16384} and all(math.isfinite(off) for off in seen.values())
    assert capsys.readouterr().out.count("tokens") == 3

    rng = np.random.default_rng(15)
    tokens, d, f = 33, 256, 160
    weight, gate, up, down = (torch.from_numpy(rng.normal(0, 0.1, s).astype(np.float32)).cuda() for s in ((d,), (f, d), (f, d), (d, f)))
    x, r = (torch.from_numpy(activations(rng, tokens, d)).cuda() for _ in range(2))
    block = example.FeedForward(weight, gate, up, down)
    got = block(x, r.clone(), block.buffers(tokens, x))
    total, n8, a8, want = torch.empty_like(r), fresh(tokens, d), fresh(tokens, f), torch.empty_like(r)
    mx8.rms_norm(x, weight, n8, residual=r, sum_out=total)
    mx8.linear(n8, block.up, a8, gate=block.gate, activation="silu")
    mx8.linear(a8, block.down, want, residual=total)
    assert torch.equal(got, want)


def test_a_matrix_follows_its_buffers_storage():
    """Weights whose storage is replaced after the Matrix was made: the product is with what the tensors hold now."""
    rng = np.random.default_rng(16)
    x, _ = matrix(activations(rng, 40, 160))
    w, _ = matrix(rng.normal(0, 0.1, (96, 160)).astype(np.float32))
    want, got = torch.empty(40, 96, device="cuda"), torch.empty(40, 96, device="cuda")
    mx8.linear(x, w, want)
    kept = w.values.data, w.scales.data
    w.values.data, w.scales.data = w.values.data.clone(), w.scales.data.clone()
    kept[0].zero_(), kept[1].zero_()
    mx8.linear(x, w, got)
    assert torch.equal(got, want) and bool(want.any())
    w.values.data = w.values.data.cpu()
    with pytest.raises(ValueError, match="CUDA"):
        mx8.linear(x, w, got)


@pytest.fixture
def large():
    """For tests of tens of GB: what they held goes back to the device, for tests that allocate without torch."""
    yield
    torch.cuda.empty_cache()


def test_the_widest_row(large):
    """2^31 - 1 columns: the last tiles' index arithmetic.  The row repeats, so each block of it is compared with a short row's."""
    cols, part = 2 ** 31 - 1, 2 ** 16
    g = torch.Generator(device="cuda").manual_seed(17)
    base = torch.randint(0, 2, (part,), generator=g, device="cuda").mul_(2).sub_(1).bfloat16()
    x = base.repeat(2 ** 31 // part)[:cols].view(1, cols)
    q = torch.full((1, 2 ** 31), 0xA5, dtype=torch.uint8, device="cuda")
    s = torch.full((mx8.scale_bytes(1, cols),), 0xA5, dtype=torch.uint8, device="cuda")
    wide, short = mx8.Matrix(q, s, 1, cols), fresh(1, part)
    mx8.quantize(base.view(1, part), short)

    def check():
        rows = q.view(-1, part)
        assert bool((rows[:-1] == short.values).all())
        assert torch.equal(rows[-1, :-1], short.values[0, :-1]) and int(rows[-1, -1]) == 0
        tiles = s.view(-1, 512)
        assert bool((tiles[:, :4] == short.scales.view(-1, 512)[0, :4]).all()) and bool((tiles[:, 4:] == 0xA5).all())

    mx8.quantize(x, wide)
    check()
    back = torch.full((1, cols), 7.0, dtype=torch.bfloat16, device="cuda")
    mx8.dequantize(wide, back)
    assert torch.equal(back, x)
    q.fill_(0xA5), s.fill_(0xA5)
    # The mean of 2^31 - 1 ones is 1 in fp32, sums of up to 2^23 of them are exact, and so is y = x.
    mx8.rms_norm(x, torch.ones(cols, device="cuda"), wide, sum_out=back.zero_(), eps=0.0)
    check()
    assert torch.equal(back, x)


@pytest.mark.parametrize("rows,cols", [(2 ** 31 - 1, 1), (2 ** 31 - 2 ** 15, 2)])
def test_rms_norm_of_the_most_rows(large, rows, cols):
    """Rows whose loop steps past 2^31: the kernels' row indices wrap there if they are signed."""
    room = 16
    sign = torch.randint(0, 2, (2 ** 16 * cols,), generator=torch.Generator(device="cuda").manual_seed(18), device="cuda").mul_(2).sub_(1)
    x = sign.half().view(-1, cols).repeat(2 ** 15, 1)[:rows]
    total = torch.zeros(rows, cols, dtype=torch.float16, device="cuda")
    q = torch.full((rows, room), 0xA5, dtype=torch.uint8, device="cuda")
    s = torch.full((mx8.scale_bytes(rows, cols),), 0xA5, dtype=torch.uint8, device="cuda")
    mx8.rms_norm(x, torch.ones(cols, device="cuda"), mx8.Matrix(q, s, rows, cols), sum_out=total, eps=0.0)
    assert torch.equal(total, x)
    # Signs over a mean square of 1: 256 in E4M3 under the scale 2^-8.
    for c in range(cols):
        assert bool((q[:, c] == torch.where(x[:, c] > 0, 0x78, 0xF8)).all())
    assert not bool(q[:, cols:].any())
    words = s.view(torch.int32)
    words = words.view(-1, 32, 4).transpose(1, 2).reshape(-1)  # by row
    assert bool((words[:rows] == 119).all())
    assert bool((words[rows:] == -0x5A5A5A5B).all())


# Bounds on an activation's relative error in fp32, in units of 2^-24: what its polynomial's fit, roundings and special
# functions add up to (the fit 2, ex2 and rcp 4 each, at most 15 for sums and products), and the rounding of the
# exponential's argument, up to three halves of a unit of it and one e-fold per unit.
ACTIVATIONS = {
    "gelu": (13.0, lambda x: 0.5 * x * torch.erfc(-x / math.sqrt(2)), lambda x: 25 + 1.5 * x * x),
    "silu": (80.0, lambda x: x * torch.sigmoid(x), lambda x: 8 + 2 * x.abs())}


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("rows,gated", [(1, False), (300, False), (2600, False), (3, True), (1200, True)])
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
def test_activations_are_relatively_exact(act, rows, gated, out_type):
    """Prescribed pre-activations (weights of zeros and a bias): the whole range of x, small results included."""
    reach, define64, bound = ACTIVATIONS[act]
    n = 1024
    at = torch.linspace(-reach, reach, n, device="cuda")
    at[:6] = torch.tensor([0.0, 1e-30, -1e-30, -1e-4, math.inf, math.nan])
    zeros = fresh(n, 64)
    mx8.quantize(torch.zeros(n, 64, device="cuda"), zeros)
    x, out = fresh(rows, 64), torch.empty(rows, n, dtype=TYPES[out_type], device="cuda")
    mx8.quantize(torch.ones(rows, 64, device="cuda"), x)
    if gated:
        mx8.linear(x, zeros, out, bias=torch.full((n,), 1.5, device="cuda"), gate=zeros, gate_bias=at, activation=act)
    else:
        mx8.linear(x, zeros, out, bias=at, activation=act)
    want = define64(at.double()) * (1.5 if gated else 1)
    assert bool((out[:, 4] == math.inf).all()) and bool(out[:, 5].isnan().all())
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[4:6] = False
    off, want, x64 = (out.double() - want).abs()[:, keep], want[keep], at.double()[keep]
    tol = want.abs() * ((bound(x64) + 1) * 2.0 ** -24 + HALF_ULP[out_type]) + TINY[out_type]
    assert bool((off <= tol).all()), float((off / tol).max())


def test_calls_without_a_stream_are_ordered_with_torchs_current_one():
    rng = np.random.default_rng(19)
    x = torch.from_numpy(activations(rng, 60, 256)).cuda()
    w, _ = matrix(rng.normal(0, 0.1, (96, 256)).astype(np.float32))
    want8, want = fresh(60, 256), torch.empty(60, 96, device="cuda")
    x.mul_(-2.0), mx8.rms_norm(x, torch.ones(256, device="cuda"), want8), mx8.linear(want8, w, want)
    x.div_(-2.0)
    got8, got, ones = fresh(60, 256), torch.empty(60, 96, device="cuda"), torch.ones(256, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # some 10 ms, in which calls on another stream would be done
        x.mul_(-2.0)
        mx8.rms_norm(x, ones, got8)
        mx8.linear(got8, w, got)
        kept = got.clone()
    side.synchronize()
    assert torch.equal(kept, want) and torch.equal(got8.values, want8.values)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mx8.rms_norm(x, ones, got8)
        mx8.linear(got8, w, got)
    got.zero_()
    graph.replay()
    assert torch.equal(got, want)


@pytest.mark.parametrize("tokens", [1, 33, 128, 200])
def test_the_examples_buffers_serve_smaller_batches(tokens):
    import importlib.util
    from pathlib import Path
    spec = importlib.util.spec_from_file_location("mx8_feed_forward", Path(__file__).resolve().parents[1] / "examples" / "mx8_feed_forward.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    rng = np.random.default_rng(20)
    d, f = 160, 224
    block = example.FeedForward(*(torch.from_numpy(rng.normal(0, 0.1, s).astype(np.float32)).cuda() for s in ((d,), (f, d), (f, d), (d, f))))
    x, r = (torch.from_numpy(activations(rng, tokens, d)).cuda() for _ in range(2))
    buffers = block.buffers(200, x)
    block(*(torch.from_numpy(activations(rng, 200, d)).cuda() for _ in range(2)), buffers)  # leaves other rows in them
    assert torch.equal(block(x, r.clone(), buffers), block(x, r.clone(), block.buffers(tokens, x)))


# -------------------------------------------------------------------------------- several turns of the row kernels' loops
#
# More rows than the blocks that are launched take at once, so that each block comes round again: with the next row's loads,
# the exchange of sums and the staging buffers of the turn before.  Neighbouring rows differ in size by powers of two, so that a
# sum or a scale of another row shows.

def scale_byte64(a):
    """Scale bytes of blocks whose largest magnitudes are `a` (float64, finite)."""
    mantissa, power = torch.frexp(a)
    e = (power - 9 + (mantissa > 0.875).int()).clamp(min=-127)
    return torch.where(a > 0, e + 127, torch.zeros_like(e))


def blocks_gpu(v):
    out = torch.zeros(v.shape[0], -(-v.shape[1] // 32) * 32, dtype=torch.float64, device="cuda")
    out[:, : v.shape[1]] = v
    return out.view(v.shape[0], -1, 32)


def bytes_gpu(m):
    return m.scales[torch.from_numpy(scale_index(m.rows, m.cols)).cuda()].int()


def expand(byte, cols):
    return torch.exp2(byte.double() - 127).repeat_interleave(32, dim=1)[:, :cols]


def spread_rows(g, rows, cols, dtype, pad=0):
    """Activations, each row times its own power of two, in a view `pad` wider than the row."""
    v = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(0.8 * torch.randn(cols, generator=g, device="cuda"))
    v *= torch.exp2(torch.randint(-5, 6, (rows, 1), generator=g, device="cuda").float())
    store = torch.full((rows, cols + pad), 7.0, dtype=dtype, device="cuda")
    store[:, :cols] = v
    return store[:, :cols]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(9000, 4096), (9000, 4095), (170000, 100), (90000, 200)])
def test_quantize_many_rows(dtype, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = spread_rows(g, rows, cols, TYPES[dtype])
    out = fresh(rows, cols)
    mx8.quantize(x, out)
    v = x.double()
    byte = scale_byte64(blocks_gpu(v).abs().amax(-1))
    assert torch.equal(bytes_gpu(out), byte.int())
    scale = expand(byte, cols)
    # Nearest multiple of the step of the value's binade (of the subnormals' below 2^-6), ties to even.
    step = torch.exp2((torch.frexp(v / scale)[1] - 1).clamp(min=-6).double() - 3)
    assert torch.equal(decode_gpu(out), torch.round(v / scale / step) * step * scale)
    assert not bool(out.values[:, cols:].any())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols,pad", [(9000, 4096, 0), (9000, 4095, 0), (9000, 4090, 3), (200000, 133, 1)])
def test_dequantize_many_rows(dtype, rows, cols, pad):
    g = torch.Generator(device="cuda").manual_seed(rows + cols + 1)
    m = fresh(rows, cols)
    m.values.copy_(torch.randint(0, 127, m.values.shape, generator=g, device="cuda"))
    m.values.bitwise_or_(torch.randint(0, 2, m.values.shape, generator=g, device="cuda").to(torch.uint8) << 7)
    m.scales.copy_(torch.randint(105, 130, m.scales.shape, generator=g, device="cuda"))
    store = torch.full((rows, cols + pad), 7.0, dtype=TYPES[dtype], device="cuda")
    mx8.dequantize(m, store[:, :cols])
    assert torch.equal(store[:, :cols], decode_gpu(m).float().to(TYPES[dtype]))  # exact in fp32
    assert bool((store[:, cols:] == 7.0).all())


MANY_ROWS = [(60000, 100), (60000, 200), (60000, 256), (20000, 768), (9000, 4096), (9000, 4095), (5000, 12001), (4000, 16384), (1500, 16401)]


@pytest.mark.parametrize("dtype,rdtype", [("bf16", "f32"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("rows,cols", MANY_ROWS)
@pytest.mark.parametrize("pad,in_place", [(0, False), (3, True)])
def test_rms_norm_many_rows(dtype, rdtype, rows, cols, pad, in_place):
    g = torch.Generator(device="cuda").manual_seed(rows + cols + 2)
    x, r = spread_rows(g, rows, cols, TYPES[dtype], pad), spread_rows(g, rows, cols, TYPES[rdtype], pad)
    w = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
    want = (x.float() + r.float()).to(TYPES[rdtype])
    h = x.double() + r.double()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-5) * w.double()
    total = r if in_place else torch.empty_like(r)
    out = fresh(rows, cols)
    mx8.rms_norm(x, w, out, residual=r, sum_out=total, eps=1e-5)
    assert torch.equal(total, want)
    if pad and in_place:
        assert bool((r.as_strided((rows, pad), (cols + pad, 1), cols) == 7.0).all())
    # `check_mx8` on the GPU; h is rounded to fp32 once before it is squared and scaled.
    slack = norm_slack(cols) * y.abs()
    a, da, byte = blocks_gpu(y).abs().amax(-1), blocks_gpu(slack).amax(-1), bytes_gpu(out)
    assert bool(((byte >= scale_byte64(a - da)) & (byte <= scale_byte64(a + da))).all())
    scale = expand(byte, cols)
    power = torch.frexp((y.abs() / scale).clamp(min=2.0 ** -6))[1] - 1
    tol = scale * torch.exp2(power.double() - 4) * (1 + 1e-12) + 2 * slack
    off = (decode_gpu(out) - y).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    assert not bool(out.values[:, cols:].any())


def test_the_example_is_as_near_to_fp32_as_its_format():
    """The block's update in MX8 against fp32.  A rounding to E4M3 is off by 0.026 of the value, root mean square: half a step,
    at most 2^-4 of its binade's lower end, evenly spread (over the root of 3) and averaged over the binade (1.44).  n, G, U, a
    and D are five such roundings; n's reaches the update through both factors of the gated product, and SiLU's slope makes
    the gate's share up to 1.5 times as large: sqrt(1.5 0.037^2 + 0.037^2 + 2 0.026^2) = 0.069.  Half as much again is allowed."""
    import importlib.util
    from pathlib import Path
    spec = importlib.util.spec_from_file_location("mx8_feed_forward", Path(__file__).resolve().parents[1] / "examples" / "mx8_feed_forward.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    for tokens, off in example.main(512, 1500):
        assert off < 0.104, (tokens, off)
