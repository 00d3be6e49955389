"""Rotary positions and attention on the GPU against their definitions in 64 bits.

Tolerances are bounds on the kernels' arithmetic, element by element: fp32 sums and products, the documented
error of the exponentials, the rounding of softmax's numerators and the one of the output (`attend_slack`,
`rotary_slack`).
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from laya_cuda import attention  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {name: torch.finfo(t).eps / 2 for name, t in TYPES.items()}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64)


# -------------------------------------------------------------------------------- rotary

def frequencies(dims, theta, scaling, factor, length, low, high):
    k = torch.arange(dims // 2, dtype=torch.float64)
    if scaling == "ntk":
        theta = theta * factor ** (dims / (dims - 2))
    f = theta ** (-2 * k / dims)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        keep = ((length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f.cuda()


def rotate(x, positions, dims, interleaved, f, magnitude, backward):
    """The definition, and the sum of the magnitudes of each result's two products."""
    w = positions.double()[:, None, None] * f
    cos, sin = magnitude * torch.cos(w), magnitude * torch.sin(w) * (-1 if backward else 1)
    k = torch.arange(dims // 2, device="cuda")
    first, second = (2 * k, 2 * k + 1) if interleaved else (k, k + dims // 2)
    out, size = x.double().clone(), x.double().abs()
    a, b = x[..., first].double(), x[..., second].double()
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = abs(magnitude) * (a.abs() + b.abs())
    return out, size


def rotary_slack(want, size, dtype):
    # Cosine and sine: the reduced angle (at most pi) rounded to fp32, the angle itself 2^-24 turns off for far positions, two
    # units of sincospif: below 2^-20 in all, of |a| + |b|.  Three roundings in fp32, one to the type.
    return 1.01 * HALF[dtype] * want.abs() + (2.0 ** -20 + 4 * 2.0 ** -24) * size + TINY[dtype]


def check_rotary(x, got, positions, dtype, dims, interleaved=False, theta=10000.0, scaling="none", factor=1.0, length=0.0,
                 low=1.0, high=32.0, magnitude=1.0, backward=False):
    f = frequencies(dims, theta, scaling, factor, length, low, high)
    want, size = rotate(x, positions, dims, interleaved, f, magnitude, backward)
    error = (got.double() - want).abs() - rotary_slack(want, size, dtype)
    assert error.max().item() <= 0 if error.numel() else True
    assert torch.equal(got[..., dims:], x[..., dims:])


def heads(g, tokens, n, dim, dtype, pad=0, offset=0):
    """A [tokens][n][dim] view of a wider buffer of sevens."""
    store = torch.full((tokens * (n * dim + pad) + offset + 16,), 7.0, dtype=TYPES[dtype], device="cuda")
    view = store[offset: offset + tokens * (n * dim + pad)].view(tokens, n * dim + pad)[:, : n * dim].unflatten(1, (n, dim))
    view.copy_(randn(g, tokens, n, dim))
    return view, store


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,n,n_k,dim,dims", [(1, 12, 12, 64, 64), (3, 1, 1, 2, 2), (77, 16, 4, 80, 32), (33, 5, 1, 40, 20), (130, 3, 2, 128, 128),
                                                  (9, 2, 2, 96, 50), (300, 32, 8, 128, 64), (2, 2, 1, 600, 512), (1, 1, 1, 7, 6)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (1, 1), (24, 8)])
def test_rotary_is_the_definition(dtype, interleaved, tokens, n, n_k, dim, dims, pad, offset):
    g = generator(tokens * 1000 + dims)
    (q, q_store), (k, _) = heads(g, tokens, n, dim, dtype, pad, offset), heads(g, tokens, n_k, dim, dtype, pad, offset)
    positions = torch.randint(0, 5000, (tokens,), generator=g, device="cuda")
    q_out, k_out = (heads(g, tokens, h, dim, dtype, pad, offset) for h in (n, n_k))
    kept = q_store.clone()
    attention.rotary(q, positions, q_out[0], k=k, k_out=k_out[0], dims=dims, interleaved=interleaved)
    check_rotary(q, q_out[0], positions, dtype, dims, interleaved)
    check_rotary(k, k_out[0], positions, dtype, dims, interleaved)
    assert torch.equal(kept, q_store)
    for view, store in (q_out, k_out):  # what lies between the rows is left as it was
        view.fill_(7.0)
        assert bool((store == 7.0).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims", [64, 24])
def test_rotary_in_place_and_one_tensor(dtype, interleaved, dims):
    g = generator(1)
    x, _ = heads(g, 50, 6, 64, dtype, 8, 0)
    before, positions = x.clone(), torch.arange(50, device="cuda", dtype=torch.int32)
    attention.rotary(x, positions, x, dims=dims, interleaved=interleaved)
    check_rotary(before, x, positions, dtype, dims, interleaved)


@pytest.mark.parametrize("scaling,factor,length,low,high", [("none", 1.0, 0, 1, 32), ("linear", 8.0, 0, 1, 32), ("ntk", 4.0, 0, 1, 32),
                                                            ("parts", 32.0, 8192, 1.0, 4.0), ("parts", 4.0, 4096, 1.0, 32.0)])
@pytest.mark.parametrize("integers", [torch.int32, torch.int64])
def test_rotary_scaled_and_far(scaling, factor, length, low, high, integers):
    g = generator(2)
    positions = torch.tensor([0, 1, 4095, 131071, 10 ** 6 + 1, 2 ** 24 + 1, 2 ** 30 + 7, 2 ** 31 - 1], device="cuda", dtype=integers)
    x, _ = heads(g, len(positions), 3, 128, "f32")
    out = torch.empty_like(x)
    how = dict(theta=500000.0, scaling=scaling, factor=factor, length=length, low=low, high=high, magnitude=1.2)
    attention.rotary(x, positions, out, **how)
    check_rotary(x, out, positions, "f32", 128, **how)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_backward_is_the_gradient(interleaved):
    g = generator(3)
    x, grad = (heads(g, 40, 4, 48, "f32")[0] for _ in range(2))
    positions = torch.arange(40, device="cuda") * 37
    how = dict(dims=32, interleaved=interleaved, scaling="linear", factor=3.0, magnitude=1.3)
    out = torch.empty_like(grad)
    attention.rotary(grad, positions, out, backward=True, **how)
    check_rotary(grad, out, positions, "f32", backward=True, **how)
    leaf = x.double().requires_grad_()
    f = frequencies(32, 10000.0, "linear", 3.0, 0, 1, 32)
    w = positions.double()[:, None, None] * f
    k = torch.arange(16, device="cuda")
    first, second = (2 * k, 2 * k + 1) if interleaved else (k, k + 16)
    a, b = leaf[..., first], leaf[..., second]
    turned = torch.cat([1.3 * (a * w.cos() - b * w.sin()), 1.3 * (a * w.sin() + b * w.cos()), leaf[..., 32:]], -1)
    order = torch.cat([first, second, torch.arange(32, 48, device="cuda")])
    turned.backward(grad.double()[..., order])
    # against the formula's gradient, and against a difference of the operator's own results (it is linear)
    bound = rotary_slack(leaf.grad, 1.3 * 2 * grad.double().abs().amax(-1, keepdim=True), "f32")
    assert ((out.double() - leaf.grad).abs() <= bound).all()
    d = randn(g, *x.shape)
    moved, still, shifted = torch.empty_like(x), torch.empty_like(x), (x.double() + d).float()
    attention.rotary(shifted, positions, moved, **how)
    attention.rotary(x, positions, still, **how)
    left = ((moved.double() - still.double()) * grad.double()).sum()
    right = (out.double() * (shifted.double() - x.double())).sum()
    scale = ((moved.double().abs() + still.double().abs() + shifted.double().abs()) * grad.double().abs()).sum() * 1.3 * 4
    assert abs(left - right) <= scale * 2.0 ** -19


@pytest.mark.parametrize("tokens,heads,strides", [(1, 3, dict(x_token=64, out_token=4096)), (5, 1, dict(x_head=64, out_head=128)), (1, 1, dict(x_token=0, x_head=0, out_token=7, out_head=9))])
def test_rotary_in_place_asks_nothing_of_a_single_dimensions_stride(tokens, heads, strides):
    import ctypes as ct
    from laya_cuda import _lib
    x = randn(generator(6), tokens, heads, 64).float()
    before, positions = x.clone(), torch.arange(3, 3 + tokens, device="cuda")
    args = _lib.Rotary(tokens=tokens, head_dim=64, dims=64, dtype=0, positions=positions.data_ptr(), positions_64=1, theta=10000.0, factor=1.0, magnitude=1.0)
    args.part[0] = _lib.Heads(**{**dict(x=x.data_ptr(), x_token=heads * 64, x_head=64, out=x.data_ptr(), out_token=heads * 64, out_head=64, heads=heads), **strides})
    torch.cuda.synchronize()
    _lib.check(_lib.load().laya_op_rotary(ct.byref(args), None))
    torch.cuda.synchronize()
    check_rotary(before, x, positions, "f32", 64)


def test_rotary_of_many_tokens():
    g = generator(4)
    x, _ = heads(g, 70001, 2, 32, "bf16")
    out, positions = torch.empty_like(x), torch.arange(70001, device="cuda")
    attention.rotary(x, positions, out)
    check_rotary(x, out, positions, "bf16", 32)


def test_rotary_keeps_infinities_and_nan_to_their_pairs():
    g = generator(5)
    x, _ = heads(g, 4, 2, 64, "bf16")
    x[1, 0, 3], x[2, 1, 40] = math.nan, math.inf
    out, positions = torch.empty_like(x), torch.arange(4, device="cuda") + 1
    attention.rotary(x, positions, out)
    bad = ~out.isfinite()
    want = torch.zeros_like(bad)
    want[1, 0, [3, 35]] = want[2, 1, [8, 40]] = True
    assert torch.equal(bad, want)


# -------------------------------------------------------------------------------- attention: the definition

def see(n, m, causal, left, right, prefix, doc_q, doc_k):
    p, j = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")
    out = torch.ones(n, m, dtype=torch.bool, device="cuda")
    if causal:
        out &= j <= p
    if left >= 0:
        out &= j >= p - left
    if right >= 0:
        out &= j <= p + right
    if doc_q is not None:
        out &= doc_q[:, None] == doc_k[None]
    return out | (j < prefix)


def define(s):
    """out and lse in 64 bits, and bounds on their errors."""
    q, k, v, how = s["q"], s["k"], s["v"], s["how"]
    dtype, h, group = s["dtype"], q.shape[1], q.shape[1] // k.shape[1]
    dim, cap, scale = q.shape[2], how.get("cap", 0.0), how.get("scale", 1 / math.sqrt(q.shape[2]))
    left, right = how.get("window") or (-1, -1)
    out, lse = torch.full(q.shape, math.nan, dtype=torch.float64, device="cuda"), torch.full(q.shape[:2], math.nan, dtype=torch.float64, device="cuda")
    out_slack, lse_slack = torch.zeros_like(out), torch.zeros_like(lse)
    k_starts, k_lengths = (s["k_starts"], s["k_lengths"]) if s["k_starts"] is not None else (s["starts"], s["lengths"])
    for b, (start, n, k_start, m) in enumerate(zip(s["starts"], s["lengths"], k_starts, k_lengths)):
        if n == 0:
            continue
        rows, keys = slice(start, start + n), slice(k_start, k_start + m)
        doc = how.get("documents")
        doc_k = how.get("k_documents", doc)
        visible = see(n, m, how.get("causal", False), left, right, s["prefix"][b] if s["prefix"] else 0,
                      None if doc is None else doc[rows], None if doc is None else doc_k[keys])
        p, j = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")
        for head in range(h):
            qs, ks, vs = q[rows, head].double(), k[keys, head // group].double(), v[keys, head // group].double()
            x = qs @ ks.T * scale
            # fp32: the sum of dim exact products (an error of 2^-24 for each addition, of the products' magnitudes), then
            # a few roundings; the cap is exact to 2^-21 of itself.
            ds = (dim + 8) * 2.0 ** -24 * (qs.abs() @ ks.abs().T) * abs(scale)
            if cap:
                x = cap * torch.tanh(x / cap)
                ds = ds + cap * 2.0 ** -21
            if "slopes" in how:
                bias = -how["slopes"][head].double() * (p - j).abs()
                x = x + bias
                ds = ds + 4 * 2.0 ** -24 * bias.abs()
            if "distance_bias" in how:
                t = how["distance_bias"][head].double()
                reach = t.numel() // 2
                bias = t[(j - p).clamp(-reach, reach) + reach]
                x = x + bias
                ds = ds + 4 * 2.0 ** -24 * torch.where(bias.isfinite(), bias.abs(), torch.zeros_like(bias))
            ds = ds + 8 * 2.0 ** -24 * x.abs()
            x = torch.where(visible, x, torch.full_like(x, -math.inf))
            top = x.amax(1, keepdim=True) if m else torch.full((n, 1), -math.inf, dtype=torch.float64, device="cuda")
            empty = top == -math.inf
            e = torch.exp(x - torch.where(empty, torch.zeros_like(top), top))
            total = e.sum(1, keepdim=True)
            w = e / torch.where(empty, torch.ones_like(total), total)
            vs = torch.where(visible.any(0)[:, None], vs, torch.zeros_like(vs)) if m else vs
            # a hidden value that is not finite has no part in the sum
            clean = torch.where(vs.isfinite(), vs, torch.zeros_like(vs))
            y = w @ clean
            poison = (visible & (w > 0)).double() @ (~vs.isfinite()).double() > 0
            out[rows, head] = torch.where(poison, torch.full_like(y, math.nan), y)
            lse[rows, head] = torch.where(empty, top, top + torch.log(torch.where(empty, torch.ones_like(total), total))).squeeze(1)
            ds = torch.where(visible & x.isfinite(), ds, torch.zeros_like(ds))
            # Each weight is off by its score's error, the exponential's 2^-13 and one rounding to the type, numerator only; below the
            # smallest numbers of the type by 2^-32 of the largest (float16).  fp32 sums over m keys.
            rel = HALF[dtype] + 2.0 ** -12 + (m / 16 + 64) * 2.0 ** -24
            spread = (w * ds).sum(1, keepdim=True)
            out_slack[rows, head] = ((w * ds) @ clean.abs() + (rel + spread) * (w @ clean.abs()) + 2.0 ** -31 * clean.abs().sum(0)
                                     + 1.01 * HALF[dtype] * y.abs() + TINY[dtype])
            lse_slack[rows, head] = (spread.squeeze(1) + 2.0 ** -12 + (m / 16 + 64) * 2.0 ** -24
                                     + 4 * 2.0 ** -24 * torch.where(empty, torch.zeros_like(top), top.abs() + 1).squeeze(1))
    return out, lse, out_slack, lse_slack


def problem(seed, queries, keys=None, heads=4, kv_heads=2, dim=64, dtype="bf16", gap=0, room=0, prefix=None, **how):
    """`keys` None: self-attention on slices of one buffer; else a cache, `room` rows more than keys apart."""
    g = generator(seed)
    s = {"dtype": dtype, "how": how, "prefix": prefix, "lengths": queries, "k_starts": None, "k_lengths": None}
    s["starts"] = [gap + sum(queries[:b]) + gap * b for b in range(len(queries))]
    rows = sum(queries) + gap * (len(queries) + 1)
    if keys is None:
        packed = randn(g, rows, heads + 2 * kv_heads, dim).to(TYPES[dtype])
        s["q"], s["k"], s["v"] = packed[:, :heads], packed[:, heads: heads + kv_heads], packed[:, heads + kv_heads:]
    else:
        s["q"] = randn(g, rows, heads, dim).to(TYPES[dtype])
        s["k_lengths"] = keys
        s["k_starts"] = [sum(keys[:b]) + room * b for b in range(len(keys))]
        s["k"], s["v"] = (randn(g, sum(keys) + room * len(keys), kv_heads, dim).to(TYPES[dtype]) for _ in range(2))
    s["q"] *= 1.5
    return s


def run(s, out=None, lse=None, **other):
    out = torch.full(s["q"].shape, 7.0, dtype=s["q"].dtype, device="cuda") if out is None else out
    lse = torch.full(s["q"].shape[:2], 7.0, device="cuda") if lse is None else lse
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    k = {} if s["k_starts"] is None else {"k_starts": ints(s["k_starts"]), "k_lengths": ints(s["k_lengths"])}
    if s["prefix"]:
        k["prefix"] = ints(s["prefix"])
    k.setdefault("max_queries", max(s["lengths"], default=0))
    k.setdefault("max_keys", max(s["k_lengths"] if s["k_lengths"] is not None else s["lengths"], default=0))
    attention.attend(s["q"], s["k"], s["v"], out, ints(s["starts"]), ints(s["lengths"]), lse=lse, err=err, **{**k, **s["how"], **other})
    assert err.item() == 0
    return out, lse


def check(s, got=None):
    out, lse = got or run(s)
    want, want_lse, slack, lse_slack = define(s)
    mine = ~want_lse.isnan()  # rows of a sequence
    assert bool((out[~mine] == 7.0).all()) and bool((lse[~mine] == 7.0).all()), "rows outside the sequences were written"
    want, got = want[mine], out[mine].double()
    assert torch.equal(want.isnan(), ~got.isfinite() | want.isnan() & got.isnan())
    error = torch.where(want.isnan(), torch.zeros_like(want), (got - want).abs() - slack[mine])
    assert error.numel() == 0 or error.max().item() <= 0, (error.max().item(), int((error > 0).sum()), error.numel())
    nothing = want_lse[mine] == -math.inf
    assert torch.equal(lse[mine] == -math.inf, nothing)
    assert not got[nothing].any()
    error = torch.where(nothing, torch.zeros_like(want_lse[mine]), (lse[mine].double() - want_lse[mine]).abs() - lse_slack[mine])
    error = error[~error.isnan()]
    assert error.numel() == 0 or error.max().item() <= 0, error.max().item()
    return out, lse


# -------------------------------------------------------------------------------- attention: sizes, layouts, types

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 12, 64), (4, 2, 128), (6, 2, 96), (7, 1, 72), (8, 1, 8), (3, 3, 40), (16, 1, 128), (128, 1, 16), (5, 5, 120)])
@pytest.mark.parametrize("causal", [False, True])
def test_self_attention(dtype, heads, kv_heads, dim, causal):
    check(problem(dim, [1, 300, 7, 128, 129, 64], heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, causal=causal))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 12, 64), (32, 8, 128), (7, 1, 80), (16, 1, 96), (1, 1, 128), (130, 65, 64)])
@pytest.mark.parametrize("queries,keys", [([1], [1]), ([1], [77]), ([1, 1, 1], [1, 128, 1000]), ([5, 1, 3], [5, 129, 2049]), ([24, 200], [4099, 700]),
                                          ([1], [20000]), ([1] * 40, [300 + 7 * b for b in range(40)])])
def test_a_cache(dtype, heads, kv_heads, dim, queries, keys):
    check(problem(len(queries), queries, keys, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, room=5, causal=True))


@pytest.mark.parametrize("queries,keys", [([0], [5]), ([3], [0]), ([0, 4, 0], [0, 9, 3]), ([9], [4]), ([300], [20]), ([200, 3], [100, 0]), ([], [])])
@pytest.mark.parametrize("causal", [False, True])
def test_empty_and_short_key_sequences(queries, keys, causal):
    check(problem(3, queries, keys, causal=causal, room=2, gap=1))


def test_no_keys_at_all():
    s = problem(3, [3, 200], [0, 0])
    assert s["k"].shape[0] == 0
    check(s)


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_between_and_behind_the_sequences_are_left(dim):
    check(problem(4, [130, 5, 260], gap=3, dim=dim, causal=True))


@pytest.mark.parametrize("dim", [64, 96])
def test_layouts(dim):
    """Heads outermost, rows of a wider buffer, and an `out` inside one."""
    s = problem(5, [200, 31], heads=4, kv_heads=4, dim=dim, causal=True)
    for name in ("q", "k", "v"):
        t = s[name]
        wide = torch.full((t.shape[1] + 1, t.shape[0], dim + 8), 3.0, dtype=t.dtype, device="cuda")
        wide[:-1, :, :dim] = t.transpose(0, 1)
        s[name] = wide[:-1, :, :dim].transpose(0, 1)
    store = torch.full((s["q"].shape[0], 6, dim + 16), 7.0, dtype=s["q"].dtype, device="cuda")
    out = store[:, 1:5, 8: dim + 8]
    check(s, run(s, out=out))
    out.fill_(7.0)
    assert bool((store == 7.0).all())


def test_bounds_above_and_below_the_lengths():
    s = problem(6, [40, 300], causal=True)
    for bounds in (dict(max_queries=340, max_keys=340), dict(max_queries=10 ** 6, max_keys=10 ** 6), dict(max_queries=None, max_keys=None)):
        got = run(s, **bounds)
        check(s, got)
    # Queries past max_queries are not computed.
    out, lse = run(s, max_queries=100)
    want, want_lse, slack, lse_slack = define(s)
    assert ((out[:140].double() - want[:140]).abs() <= slack[:140]).all() and ((lse[:140].double() - want_lse[:140]).abs() <= lse_slack[:140]).all()
    assert bool((out[140:] == 7.0).all()) and bool((lse[140:] == 7.0).all())
    # max_keys only shapes the launch.
    check(s, run(s, max_keys=3))


def test_offsets_past_32_bits():
    """Keys and values of a cache whose later sequences start more than 2^32 bytes in, and 2^31 values."""
    rows, dim, kv = 2 ** 31 // (128 * 4) + 5000, 128, 4
    k, v = (torch.zeros(rows, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    s = problem(7, [1, 1, 6], [4000, 77, 900], heads=8, kv_heads=kv, dim=dim, causal=True)
    at = [rows - 4000, 10, rows - 4900]
    for b, (start, m) in enumerate(zip(s["k_starts"], s["k_lengths"])):
        k[at[b]: at[b] + m], v[at[b]: at[b] + m] = s["k"][start: start + m], s["v"][start: start + m]
    s["k"], s["v"], s["k_starts"] = k, v, at
    check(s)


@pytest.mark.parametrize("token,head", [(3, 2), (2, 3), (5, 2), (2, 7)])
def test_heads_between_one_another(token, head):
    """Strides of `token` and `head` heads: neither dimension within a step of the other, and no two the same."""
    s = problem(70, [2, 1] if head < token else [1, 1], heads=2 if token != 5 else 3, kv_heads=1, dim=64, causal=True)
    rows, heads = s["q"].shape[:2]
    assert len({i * token + j * head for i in range(rows) for j in range(heads)}) == rows * heads
    store = torch.full(((rows - 1) * token + (heads - 1) * head + 1, 64), 7.0, dtype=s["q"].dtype, device="cuda").view(-1)
    out = store.as_strided((rows, heads, 64), (token * 64, head * 64, 1))
    check(s, run(s, out=out))
    positions = torch.arange(rows, device="cuda")
    before = s["q"].clone()
    attention.rotary(s["q"], positions, out)
    check_rotary(before, out, positions, "bf16", 64)


# -------------------------------------------------------------------------------- attention: masks, caps, biases

def documents(lengths, mean, seed, order=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in lengths:
        ids = torch.cumsum((torch.rand(n, generator=g) < 1 / mean).long(), 0)
        out.append(ids if not order else torch.randint(0, 3, (n,), generator=g))
    return torch.cat(out).to(torch.int32).cuda()


MASKS = [dict(), dict(causal=True), dict(window=(0, 0)), dict(window=(17, 100)), dict(window=(-1, 3)), dict(window=(64, -1)), dict(causal=True, window=(200, -1)),
         dict(causal=True, window=(-1, 5))]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("prefix", [None, [1, 100, 5, 400]])
@pytest.mark.parametrize("doc", ["none", "runs", "mixed"])
@pytest.mark.parametrize("dim", [64, 128])
def test_masks(mask, prefix, doc, dim):
    lengths = [260, 515, 1, 390]
    if doc != "none":
        mask = {**mask, "documents": documents(lengths, 60, 1, doc == "mixed")}
    check(problem(8, lengths, heads=3, kv_heads=1, dim=dim, prefix=prefix, **mask))


@pytest.mark.parametrize("doc", [None, 40])
@pytest.mark.parametrize("mask", [dict(causal=True), dict(window=(100, 20)), dict()])
@pytest.mark.parametrize("queries", [[2, 1, 7], [150, 1, 64]])
def test_masks_over_a_cache(mask, doc, queries):
    keys = [300, 4000, 1290]
    if doc:
        k_documents = documents(keys, doc, 2)
        starts = [0, 300, 4300]
        mask = {**mask, "k_documents": k_documents, "documents": torch.cat([k_documents[a + m - n: a + m] for a, m, n in zip(starts, keys, queries)])}
    check(problem(9, queries, keys, heads=8, kv_heads=2, dim=128, prefix=[20, 1000, 0], **mask))


BIASES = [dict(cap=30.0), dict(cap=0.5), dict(slopes=True), dict(distance_bias=128), dict(distance_bias=0), dict(distance_bias=1000), dict(cap=20.0, slopes=True),
          dict(cap=50.0, distance_bias=16)]


def with_bias(how, heads, seed=0):
    how = dict(how)
    if "slopes" in how:
        how["slopes"] = torch.exp2(-8 * torch.arange(1, heads + 1, device="cuda") / heads)
    if "distance_bias" in how:
        how["distance_bias"] = randn(generator(seed), heads, 2 * how["distance_bias"] + 1).float()
    return how


@pytest.mark.parametrize("how", BIASES)
@pytest.mark.parametrize("mask", [dict(), dict(causal=True), dict(window=(90, 40))])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (6, 2, 128)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_caps_and_biases(how, mask, heads, kv_heads, dim, dtype):
    check(problem(10, [300, 17, 1], heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, **with_bias(how, heads), **mask))


@pytest.mark.parametrize("how", BIASES)
@pytest.mark.parametrize("queries", [[1, 3], [20, 130]])
def test_caps_and_biases_over_a_cache(how, queries):
    check(problem(11, queries, [900, 2500], heads=14, kv_heads=2, dim=64, **with_bias(how, 14), causal=True))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("cap", [0.0, 25.0])
def test_scales(dtype, scale, cap):
    """A scale of zero, a negative one, and one that makes single keys take all the weight."""
    check(problem(12, [200, 50], dim=64, dtype=dtype, scale=scale, cap=cap, causal=True))


@pytest.mark.parametrize("value", [-math.inf, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("queries,keys", [([300], None), ([1, 3], [700, 200])])
def test_biases_that_mask(value, queries, keys):
    """Distances ruled out by the bias; with the type's lowest value everywhere the weights are equal."""
    table = torch.zeros(4, 101, device="cuda")
    table[0, :] = value
    table[1, 40:60] = value
    table[2, 0] = table[2, -1] = value
    check(problem(13, queries, keys, heads=4, kv_heads=2, distance_bias=table))


def test_scores_rising_and_falling_along_the_keys():
    """The running maximum is passed again and again, by much and by little."""
    for sign in (1, -1):
        s = problem(14, [150, 1], [3000, 2500], heads=4, kv_heads=2, dim=64, dtype="f16")
        ramp = torch.linspace(-1, 1, 5500, device="cuda", dtype=torch.float64)
        s["q"] = (s["q"].double() * 0.1 + 1).half()
        s["k"] = (s["k"].double() * 0.1 + sign * 4 * ramp[:, None, None]).half()
        check(s)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [64, 128])
def test_hidden_keys_may_hold_anything(bad, dim):
    """Rows outside the sequences, a cache's unused rows, and keys that a mask hides from some queries."""
    s = problem(15, [3, 200], [150, 420], heads=4, kv_heads=2, dim=dim, room=64, gap=2, causal=True)
    for name in ("k", "v"):
        t = s[name]
        for start, m in zip(s["k_starts"], s["k_lengths"]):
            t[start + m: start + m + 64] = bad
    check(s)
    out, lse = run(s)
    assert bool(out[s["starts"][1]: s["starts"][1] + 200].isfinite().all())
    s["v"][s["k_starts"][1] + 300, 1, 5] = bad  # seen by queries 80 and on of the second sequence
    check(s)
    lengths = [260, 300]
    s = problem(16, lengths, heads=4, kv_heads=4, dim=dim, documents=documents(lengths, 50, 3))
    hit = s["how"]["documents"][:260] == s["how"]["documents"][100]
    s["v"][:260][hit] = bad
    s["k"][:260][hit] = bad
    s["how"]["documents"] = s["how"]["documents"].clone()
    out, lse = run(s)
    clean = torch.ones(sum(lengths), dtype=torch.bool, device="cuda")
    clean[:260] = ~hit
    assert bool(out[clean].isfinite().all()) and bool(lse[clean].isfinite().all())
    want = problem(16, lengths, heads=4, kv_heads=4, dim=dim, documents=s["how"]["documents"])
    exact, _, slack, _ = define(want)
    assert ((out[clean].double() - exact[clean]).abs() <= slack[clean]).all()


def narrow_bounds(s):
    """out and lse in 64 bits, and bounds that count each rounding: exponentials to 2^-22 of themselves, a cap's polynomial up to 0.8 of the cap, with its
    roundings, to 2^-21 of its result, beyond that to 2^-21 of the cap, the logarithm to a unit in its last place."""
    u, how, (rows, heads, dim), kv = 2.0 ** -24, s["how"], s["q"].shape, s["k"].shape[1]
    cap, k_starts, k_lengths = how.get("cap", 0.0), s["k_starts"] or s["starts"], s["k_lengths"] or s["lengths"]
    out, lse = torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda"), torch.zeros(rows, heads, dtype=torch.float64, device="cuda")
    out_slack, lse_slack = torch.zeros_like(out), torch.zeros_like(lse)
    for start, n, k_start, m in zip(s["starts"], s["lengths"], k_starts, k_lengths):
        at, keys = slice(start, start + n), slice(k_start, k_start + m)
        p, j = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")
        for h in range(heads):
            q, k, v = s["q"][at, h].double(), s["k"][keys, h * kv // heads].double(), s["v"][keys, h * kv // heads].double()
            x, ds = q @ k.T / math.sqrt(dim), (dim + 8) * u * (q.abs() @ k.abs().T) / math.sqrt(dim)
            if cap:
                near = (x / cap).abs() <= 0.8
                x = cap * torch.tanh(x / cap)
                ds = ds + 2.0 ** -21 * torch.where(near, x.abs(), torch.full_like(x, cap))
            bias = torch.zeros_like(x)
            if "slopes" in how:
                bias = -how["slopes"][h].double() * (p - j).abs()
            if "distance_bias" in how:
                table = how["distance_bias"][h].double()
                bias = table[(j - p).clamp(-(len(table) // 2), len(table) // 2) + len(table) // 2]
            x = x + bias
            if how.get("causal"):
                x = torch.where(j <= p, x, torch.full_like(x, -math.inf))
            top, w, full = x.amax(1), torch.softmax(x, 1), torch.logsumexp(x, 1)
            ds = torch.where(w > 0, ds + 4 * u * bias.abs() + 6 * u * (x.abs() + top[:, None].abs()), torch.zeros_like(ds))
            spread, sums = (w * ds).sum(1), 2.0 ** -21 + (m / 16 + 64) * u
            y, size = w @ v, w @ v.abs()
            out[at, h], lse[at, h] = y, full
            out_slack[at, h] = ((w * ds) @ v.abs() + (HALF[s["dtype"]] + sums + spread[:, None]) * size + 2.0 ** -31 * v.abs().sum(0)
                                + 1.01 * HALF[s["dtype"]] * y.abs() + TINY[s["dtype"]])
            lse_slack[at, h] = spread + sums + 2 * u * (math.log(m) + 10) + 6 * u * (full.abs() + top.abs() + 1)
    return out, lse, out_slack, lse_slack


@pytest.mark.parametrize("how", [dict(), dict(cap=30.0), dict(cap=2.0), dict(cap=500.0), dict(slopes=True), dict(distance_bias=50), dict(cap=20.0, slopes=True), dict(cap=50.0, distance_bias=16)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (3, 1, 128)])
@pytest.mark.parametrize("queries,keys", [([300, 129], None), ([1, 3], [1500, 200])])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_logarithms_and_caps_to_their_roundings(how, heads, kv_heads, dim, queries, keys, dtype):
    s = problem(80, queries, keys, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, causal=True, **with_bias(how, heads))
    out, lse = run(s)
    want, want_lse, slack, lse_slack = narrow_bounds(s)
    off = (lse.double() - want_lse).abs()
    assert bool((off <= lse_slack).all()), ((off / lse_slack).max().item(), off.max().item(), lse_slack.max().item())
    off = (out.double() - want).abs()
    assert bool((off <= slack).all()), (off / slack).max().item()


# -------------------------------------------------------------------------------- attention: calls

@pytest.mark.parametrize("queries,keys", [([300, 200], None), ([1, 1], [9000, 300])])
def test_the_same_each_time(queries, keys):
    s = problem(17, queries, keys, heads=16, kv_heads=4, dim=128, causal=True, cap=40.0)
    first = run(s)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, run(s)))


def test_sequences_outside_the_tensors_are_reported_and_skipped():
    s = problem(18, [40, 50, 60], [100, 200, 300], causal=True, dim=64)
    want, _ = run(s, max_queries=None, max_keys=None)  # the bounds decide how the keys are split, and so the last bits
    for name, at, value in (("starts", 1, -1), ("lengths", 1, 2 ** 30), ("k_starts", 1, 550), ("k_lengths", 1, -4), ("k_lengths", 1, 2 ** 31 - 1)):
        fields = {n: list(s[n]) for n in ("starts", "lengths", "k_starts", "k_lengths")}
        fields[name][at] = value
        out, err = torch.full_like(want, 7.0), torch.zeros(1, dtype=torch.int32, device="cuda")
        attention.attend(s["q"], s["k"], s["v"], out, ints(fields["starts"]), ints(fields["lengths"]), ints(fields["k_starts"]),
                         ints(fields["k_lengths"]), causal=True, err=err)
        assert err.item() == 4
        assert torch.equal(out[:40], want[:40]) and torch.equal(out[90:], want[90:]) and bool((out[40:90] == 7.0).all())


def test_streams_and_a_captured_graph_with_new_lengths():
    s = problem(19, [1, 1], [5000, 3000], heads=8, kv_heads=2, dim=128, causal=True)
    starts, lengths, k_starts, k_lengths = (ints(s[n]) for n in ("starts", "lengths", "k_starts", "k_lengths"))
    positions = torch.tensor([4999, 2999], device="cuda")
    q, out = torch.empty_like(s["q"]), torch.empty_like(s["q"])

    def step():
        attention.rotary(s["q"], positions, q)
        attention.attend(q, s["k"], s["v"], out, starts, lengths, k_starts, k_lengths, max_queries=1, max_keys=5000, causal=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    eager = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    out.zero_()
    graph.replay()
    assert torch.equal(out, eager)
    k_lengths.copy_(ints([1200, 2]))
    positions.copy_(torch.tensor([1199, 1], device="cuda"))
    graph.replay()
    replayed = out.clone()
    step()
    assert torch.equal(out, replayed)
    turned = {**s, "q": q, "k_lengths": [1200, 2]}
    want, _, slack, _ = define(turned)
    assert ((replayed.double() - want).abs() <= slack).all()


def test_two_calls_at_once():
    problems = [problem(20 + i, [700, 300], heads=8, kv_heads=4, dim=64, causal=True) for i in range(2)]
    want = [run(s) for s in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, stream in zip(problems, streams):
            with torch.cuda.stream(stream):
                got.append(run(s))
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(lse, want[i % 2][1])


@pytest.mark.parametrize("threads", [1, 2])
def test_calls_in_flight_together(threads):
    """Each on a stream of its own, held back until all are enqueued: tiles of both head sizes, single tokens in a quarter of a tile and over a cluster, joined
    halves.  Few CTAs each, so that those of different calls share the GPU and its SMs."""
    from concurrent.futures import ThreadPoolExecutor
    forms = [problem(72, [260, 100], heads=4, kv_heads=2, dim=64, causal=True), problem(73, [300], heads=4, kv_heads=2, dim=128, causal=True, cap=30.0),
             problem(74, [1, 1], [9000, 300], heads=8, kv_heads=2, dim=128), problem(75, [40], [700], heads=2, kv_heads=1, dim=128, causal=True),
             problem(76, [1] * 9, [200] * 9, heads=4, kv_heads=2, dim=64, causal=True), problem(77, [200, 90], heads=4, kv_heads=2, dim=64, distance_bias=randn(generator(1), 4, 41).float())]
    calls = []
    for s in forms:
        want, want_lse = check(s)
        k = {} if s["k_starts"] is None else {"k_starts": ints(s["k_starts"]), "k_lengths": ints(s["k_lengths"])}
        bounds = dict(max_queries=max(s["lengths"]), max_keys=max(s["k_lengths"] or s["lengths"]))
        calls.append(dict(args=(s["q"], s["k"], s["v"]), out=torch.empty_like(want), starts=ints(s["starts"]), lengths=ints(s["lengths"]), how={**k, **bounds, **s["how"]},
                          lse=torch.empty_like(want_lse), err=torch.zeros(1, dtype=torch.int32, device="cuda"), want=want, want_lse=want_lse,
                          others=torch.zeros((), dtype=torch.int64, device="cuda"), stream=torch.cuda.Stream()))
    torch.cuda.synchronize()
    gate = torch.cuda.Event()
    torch.cuda._sleep(40_000_000)
    gate.record()

    def enqueue(some):
        for c in some:
            c["stream"].wait_event(gate)
        for _ in range(25):
            for c in some:
                with torch.cuda.stream(c["stream"]):
                    c["out"].fill_(7.0)
                    attention.attend(*c["args"], c["out"], c["starts"], c["lengths"], lse=c["lse"], err=c["err"], **c["how"])
                    c["others"] += (c["out"] != c["want"]).sum() + (c["lse"] != c["want_lse"]).sum()

    if threads == 1:
        enqueue(calls)
    else:
        with ThreadPoolExecutor(threads) as pool:
            list(pool.map(enqueue, (calls[::2], calls[1::2])))
    torch.cuda.synchronize()
    assert [c["err"].item() for c in calls] == [0] * len(calls)
    assert [c["others"].item() for c in calls] == [0] * len(calls)


def test_pieces_join_by_their_logarithms():
    """A shared prefix and the rest of the keys, attended apart, give the whole."""
    s = problem(22, [30], [1000], heads=4, kv_heads=2, dim=64)
    want, _, slack, _ = define(s)
    parts = []
    for first, last in ((0, 333), (333, 1000)):
        parts.append(run({**s, "k_starts": [first], "k_lengths": [last - first]}))
    lse = torch.stack([p[1].double() for p in parts])
    w = torch.softmax(lse, 0)[..., None]
    joined = sum(wi * p[0].double() for wi, p in zip(w, parts))
    # Each part within its own bound, which the weights mix; the weights are off by the logarithms' errors.
    assert ((joined - want).abs() <= 3 * slack + 2.0 ** -10 * want.abs() + 2.0 ** -11).all()


# -------------------------------------------------------------------------------- attention: what decides between its ways

@pytest.mark.parametrize("heads,kv_heads,queries", [(32, 1, [1, 1]), (16, 1, [2, 1]), (33, 1, [1, 1]), (8, 8, [32, 7]), (8, 8, [33, 1]), (5, 1, [6, 2]), (128, 1, [1, 2]),
                                                    (100, 1, [2, 1])])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("how", [dict(), dict(cap=30.0), dict(slopes=True), dict(distance_bias=100)])
def test_rows_about_a_quarter_and_a_whole_tile(heads, kv_heads, queries, dim, how):
    check(problem(30, queries, [700, 133], heads=heads, kv_heads=kv_heads, dim=dim, causal=True, prefix=[3, 0], **with_bias(how, heads)))


@pytest.mark.parametrize("queries", [[1, 1], [5, 2], [200, 20]])
@pytest.mark.parametrize("window", [None, (300, 10), (0, 0)])
def test_masks_of_few_rows(queries, window):
    keys = [1500, 260]
    k_documents = documents(keys, 100, 4)
    doc = torch.cat([k_documents[a + m - n: a + m] for a, m, n in zip([0, 1500], keys, queries)])
    check(problem(31, queries, keys, heads=8, kv_heads=2, dim=64, window=window, documents=doc, k_documents=k_documents, prefix=[130, 0]))


@pytest.mark.parametrize("queries", [[1], [40]])
@pytest.mark.parametrize("mixed", [False, True])
def test_documents_of_many_steps(queries, mixed):
    """More steps of keys than are looked over ahead, with documents that come back far apart."""
    keys = [50000]
    k_documents = documents(keys, 4000, 5)
    if mixed:
        k_documents = k_documents % 3
    check(problem(32, queries, keys, heads=2, kv_heads=1, dim=64, documents=k_documents[-queries[0]:].clone(), k_documents=k_documents))


@pytest.mark.parametrize("reach,heads,kv_heads", [(3000, 2, 2), (1000, 8, 1), (128, 64, 2), (1, 6, 2)])
@pytest.mark.parametrize("queries,keys", [([300], None), ([1, 60], [3000, 200])])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_distance_biases_of_all_sizes(reach, heads, kv_heads, queries, keys, cap):
    how = with_bias(dict(distance_bias=reach), heads, reach)
    check(problem(33, queries, keys, heads=heads, kv_heads=kv_heads, dim=64, cap=cap, **how))


@pytest.mark.parametrize("scale,cap", [(0.125, 0.01), (0.125, 1e-4), (0.125, 500.0), (0.125, 1e5), (3.0, 4.0), (1.0, 1e-3), (-0.3, 5.0), (1e-3, 50.0)])
@pytest.mark.parametrize("queries,keys", [([300], None), ([1, 3], [900, 200])])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_caps_far_below_and_far_above_the_scores(scale, cap, queries, keys, dtype):
    check(problem(34, queries, keys, heads=4, kv_heads=2, dim=64, dtype=dtype, scale=scale, cap=cap, causal=True))


@pytest.mark.parametrize("sequences,kv_heads,dim", [(3, 8, 128), (6, 8, 64), (13, 8, 128), (24, 8, 64), (128, 2, 64), (129, 2, 64)])
@pytest.mark.parametrize("queries", [1, 2])
def test_single_tokens_over_caches_of_all_lengths(sequences, kv_heads, dim, queries):
    keys = [[4700, 0, 1, 4700, 129, 8200, 3000, 0, 128, 6000][b % 10] // (1 if sequences < 100 else 4) for b in range(sequences)]
    s = problem(37, [queries] * sequences, keys, heads=2 * kv_heads, kv_heads=kv_heads, dim=dim, causal=True)
    check(s)
    first = run(s, max_keys=40000)
    check(s, first)
    assert all(torch.equal(a, b) for a, b in zip(first, run(s, max_keys=40000)))


@pytest.mark.parametrize("how", [dict(), dict(causal=True), dict(distance_bias=20), dict(slopes=True), dict(window=(-1, 60))])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_sequences_of_several_tiles(how, dim):
    lengths = [[300, 0, 1, 129, 260, 64, 128, 5][b % 8] for b in range(80)]
    check(problem(38, lengths, heads=4, kv_heads=2, dim=dim, **with_bias(how, 4)))


@pytest.mark.parametrize("cap", [2e3, 1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("queries,keys", [([300], None), ([1, 3], [900, 200])])
@pytest.mark.parametrize("slopes", [False, True])
def test_a_cap_that_no_score_reaches_changes_little(cap, queries, keys, slopes):
    # |x - cap tanh(x / cap)| <= |x|^3 / (3 cap^2), and |x| is below 10: scores of 64 products with a deviation of 1.
    s = problem(36, queries, keys, heads=4, kv_heads=2, dim=64, dtype="bf16", cap=cap, causal=True, **(with_bias(dict(slopes=True), 4) if slopes else {}))
    out, lse = run(s)
    how = {k: v for k, v in s["how"].items() if k != "cap"}
    want, want_lse, slack, lse_slack = define(dict(s, how=how))
    less = 1000 / (3 * cap * cap)
    assert ((lse.double() - want_lse).abs() <= lse_slack + less).all()
    assert ((out.double() - want).abs() <= slack + 2 * less * s["v"].double().abs().max()).all()


@pytest.mark.parametrize("slope", [0.0, 1e-6, 3.0, -0.25])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,keys", [([500], None), ([1, 40], [3000, 700])])
def test_slopes_of_all_sizes(slope, causal, queries, keys):
    """Also ones that favour far keys, whose maximum the steps raise again and again."""
    check(problem(35, queries, keys, heads=2, kv_heads=2, dim=64, causal=causal, slopes=torch.full((2,), slope, device="cuda")))


def test_the_largest_documented_values():
    """Documents and prefixes at the ends of 32 bits, windows as wide as numbers go."""
    lengths = [300, 40]
    doc = torch.randint(0, 2, (340,), generator=generator(6), device="cuda").mul(2 ** 32 - 1).sub(2 ** 31).to(torch.int32)
    check(problem(36, lengths, heads=2, kv_heads=1, dim=64, documents=doc, window=(2 ** 31 - 1, 2 ** 31 - 1), prefix=[2 ** 31 - 1, -2 ** 31]))
    check(problem(36, lengths, heads=2, kv_heads=1, dim=64, causal=True, window=(2 ** 31 - 1, 0), prefix=[-5, 0]))


def test_a_wait_that_runs_out_is_reported_and_leaves_the_device_usable():
    """A valid call whose waits are limited to a nanosecond: it gives up, says so, and the next call is right."""
    from laya_cuda import _lib
    lib = _lib.load()
    for queries, keys in (([1000], None), ([1], [9000]), ([20], [9000])):
        s = problem(37, queries, keys, heads=4, kv_heads=1, dim=128, causal=True)
        out, err = torch.zeros(s["q"].shape, dtype=s["q"].dtype, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        k = {} if keys is None else {"k_starts": ints(s["k_starts"]), "k_lengths": ints(s["k_lengths"])}
        _lib.check(lib.laya_set_launch_options(1, 1))
        try:
            attention.attend(s["q"], s["k"], s["v"], out, ints(s["starts"]), ints(s["lengths"]), err=err, causal=True, **k)
            torch.cuda.synchronize()
        finally:
            _lib.check(lib.laya_set_launch_options(1, 0))
        assert err.item() == 5
        check(s)


@pytest.mark.parametrize("queries,keys,dim", [([700, 300], None, 64), ([700, 300], None, 128), ([1] * 40, [3000] * 40, 128), ([20, 1], [9000, 0], 64)])
def test_waits_that_run_out_early_and_late(queries, keys, dim):
    """Limits under which some waits run out and others do not: a call that reports nothing is right, and calls after it are."""
    from laya_cuda import _lib
    lib = _lib.load()
    s = problem(61, queries, keys, heads=8, kv_heads=2, dim=dim, causal=True)
    want, _ = check(s)
    k = {} if keys is None else {"k_starts": ints(s["k_starts"]), "k_lengths": ints(s["k_lengths"])}
    starts, lengths, out = ints(s["starts"]), ints(s["lengths"]), torch.empty_like(want)
    reported = set()
    for limit in (1, 200, 700, 2000, 5000, 15000):
        _lib.check(lib.laya_set_launch_options(1, limit))
        try:
            for _ in range(5):
                err = torch.zeros(1, dtype=torch.int32, device="cuda")
                out.fill_(7.0)
                attention.attend(s["q"], s["k"], s["v"], out, starts, lengths, max_queries=max(queries), max_keys=max(keys or queries), causal=True, err=err, **k)
                reported.add(err.item())
                assert err.item() == 5 or torch.equal(out, want)
        finally:
            _lib.check(lib.laya_set_launch_options(1, 0))
        check(s)
    assert 5 in reported and reported <= {0, 5}


# -------------------------------------------------------------------------------- attention: tiles that no key is visible to

def some_sequences(s, which):
    return {**s, **{n: [s[n][b] for b in which] for n in ("starts", "lengths", "k_starts", "k_lengths")}}


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", ["no keys", "before the first key", "a document without keys", "single tokens", "shares without keys"])
def test_thousands_of_tiles_without_a_visible_key(form, dim):
    """Their queries come from memory, not from the L2 cache, and are of no use to any product."""
    heads, how = 4, {}
    if form == "no keys":
        queries, keys = [130] * 1200, [200 if b % 50 == 7 else 0 for b in range(1200)]
    elif form == "before the first key":
        queries, keys, how = [400] * 400, [20] * 400, {"causal": True}
    elif form == "a document without keys":
        queries, keys = [130] * 1200, [64] * 1200
        other = torch.tensor([b % 50 != 7 for b in range(1200)], device="cuda").int()
        how = {"documents": other.repeat_interleave(130), "k_documents": torch.zeros(1200 * 64, dtype=torch.int32, device="cuda")}
    elif form == "single tokens":
        queries, keys, heads = [1] * 6000, [200 if b % 500 == 7 else 0 for b in range(6000)], 32
    else:  # a cluster's CTAs past the last key of a short cache
        queries, keys, heads = [1] * 4, [130, 0, 5000, 1], 16
    s = problem(60, queries, keys, heads=heads, kv_heads=2, dim=dim, **how)
    some = [b for b, m in enumerate(keys) if m and (len(keys) < 10 or b % 50 == 7)]
    part = some_sequences(s, some)
    want, want_lse, slack, lse_slack = define(part)
    mine = ~want_lse.isnan()
    nothing = torch.ones(len(s["q"]), dtype=torch.bool, device="cuda")
    for b, (start, n) in enumerate(zip(s["starts"], queries)):
        if form == "before the first key":
            nothing[start + n - 20: start + n] = False
        elif keys[b] and (form != "a document without keys" or b % 50 == 7):
            nothing[start: start + n] = False
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for i in range(4):
        flush.fill_(i)
        out, lse = run(s, **({"max_keys": 40000} if form == "shares without keys" else {}))
        assert not out[nothing].any() and bool((lse[nothing] == -math.inf).all())
        assert ((out.double() - want).abs() <= slack)[mine].all()
        empty = want_lse == -math.inf
        assert ((lse.double() - want_lse).abs() <= lse_slack)[mine & ~empty].all()


# -------------------------------------------------------------------------------- attention: values that are not finite

def same_kinds(got, want):
    """NaN for NaN, infinities for infinities of their sign."""
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf())


@pytest.mark.parametrize("queries,keys,heads", [([1], [9000], 4), ([2, 1], [9000, 700], 8), ([24], [9000], 4), ([300], [3000], 4), ([300], [400], 4)])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_visible_nan_counts_however_small_its_weight(queries, keys, heads, dim):
    """Weights below the smallest number of 32 bits, in a part of the keys that has no other."""
    s = problem(62, queries, keys, heads=heads, kv_heads=2, dim=dim)
    s["q"].fill_(1.0)
    s["k"].fill_(-120 / dim ** 0.5)
    for start in s["k_starts"]:
        s["k"][start: start + 100] = 120 / dim ** 0.5
    assert math.exp(-240) > 0 and 2 ** -149 > math.exp(-240)
    at = s["k_starts"][0] + keys[0] - 50
    s["v"][at, 1, 3] = math.nan
    out, _ = check(s)
    assert bool(out[: queries[0], heads // 2:, 3].isnan().all())


def kinds(s):
    """Which results are NaN, and which are infinities, for values that are not and weights that are all above zero."""
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    how, group = s["how"], s["q"].shape[1] // s["k"].shape[1]
    left, right = how.get("window") or (-1, -1)
    k_starts, k_lengths = (s["k_starts"], s["k_lengths"]) if s["k_starts"] is not None else (s["starts"], s["lengths"])
    for b, (start, n, k_start, m) in enumerate(zip(s["starts"], s["lengths"], k_starts, k_lengths)):
        rows, keys = slice(start, start + n), slice(k_start, k_start + m)
        doc = how.get("documents")
        doc_k = how.get("k_documents", doc)
        sees = see(n, m, how.get("causal", False), left, right, s["prefix"][b] if s["prefix"] else 0,
                   None if doc is None else doc[rows], None if doc is None else doc_k[keys]).double()
        for head in range(s["q"].shape[1]):
            v = s["v"][keys, head // group]
            nan, up, down = (sees @ t.double() > 0 for t in (v.isnan(), v.isposinf(), v.isneginf()))
            y = out[rows, head]
            y[up], y[down] = math.inf, -math.inf
            y[nan | (up & down)] = math.nan
    return out


@pytest.mark.parametrize("form", ["causal", "window", "documents", "prefix", "few rows", "single tokens"])
@pytest.mark.parametrize("heads,dim", [(2, 64), (6, 128), (4, 40)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("often", [0.002, 0.05])
def test_infinities_and_nan_are_those_of_the_visible_values(form, heads, dim, dtype, often):
    """Whatever the hidden values of the same channels are, in a mask's steps and in those past them."""
    lengths = [300, 129]
    if form == "few rows":
        s = problem(63, [40, 20], [700, 133], heads=heads, kv_heads=2, dim=dim, dtype=dtype, causal=True)
    elif form == "single tokens":
        keys = [3000, 200]
        k_documents = documents(keys, 300, 7) % 3
        s = problem(63, [2, 1], keys, heads=heads, kv_heads=2, dim=dim, dtype=dtype, documents=k_documents[torch.tensor([2998, 2999, 3199], device="cuda")].clone(),
                    k_documents=k_documents)
    else:
        how = {"causal": dict(causal=True), "window": dict(window=(70, 9)), "documents": dict(documents=documents(lengths, 40, 6)), "prefix": dict(causal=True, window=(20, -1))}[form]
        s = problem(63, lengths, heads=heads, kv_heads=2, dim=dim, dtype=dtype, prefix=[60, 7] if form == "prefix" else None, **how)
    g = generator(64)
    for value in (math.nan, math.inf, -math.inf):
        s["v"][torch.rand(s["v"].shape, generator=g, device="cuda") < often / 12] = value
    out, lse = run(s)
    want = kinds(s)
    mine = ~define(s)[1].isnan()
    assert same_kinds(out[mine].double(), want[mine])
    # Where all a row's values are finite, it is the definition's.
    clean = {**s, "v": torch.where(s["v"].isfinite(), s["v"], torch.zeros_like(s["v"]))}
    exact, exact_lse, slack, lse_slack = define(clean)
    fine = (want == 0) & mine[..., None]
    assert (out.double() - exact)[fine].abs().sub(slack[fine]).max() <= 0
    seen = mine & (exact_lse != -math.inf)
    assert (lse.double() - exact_lse)[seen].abs().sub(lse_slack[seen]).max() <= 0


@pytest.mark.parametrize("queries,keys", [([24], [9000]), ([1], [9000]), ([5, 100], [7000, 3000]), ([40], [50000])])
@pytest.mark.parametrize("heads,dim", [(2, 72), (8, 128), (4, 8)])
@pytest.mark.parametrize("mask", ["documents", "window", "prefix"])
def test_infinities_and_nan_over_split_keys(queries, keys, heads, dim, mask):
    """Hidden and visible ones in the shares of several CTAs of a cluster, and past the steps whose documents are looked over ahead."""
    how = {"window": (500, 3)} if mask == "window" else {}
    if mask != "window":
        k_documents = documents(keys, 700, 8) % (3 if mask == "documents" else 2)
        at = torch.cat([sum(keys[:b]) + m - n + torch.arange(n, device="cuda") for b, (n, m) in enumerate(zip(queries, keys))])
        how = dict(documents=k_documents[at].clone(), k_documents=k_documents)
    s = problem(81, queries, keys, heads=heads, kv_heads=2, dim=dim, prefix=[1300] * len(queries) if mask == "prefix" else None, **how)
    g = generator(82)
    for value in (math.nan, math.inf, -math.inf):
        s["v"][torch.rand(s["v"].shape, generator=g, device="cuda") < 0.25 / sum(keys)] = value
    out, lse = run(s)
    want = kinds(s)
    assert same_kinds(out.double(), want)
    clean = {**s, "v": torch.where(s["v"].isfinite(), s["v"], torch.zeros_like(s["v"]))}
    exact, exact_lse, slack, lse_slack = define(clean)
    fine = want == 0
    assert (out.double() - exact)[fine].abs().sub(slack[fine]).max() <= 0
    assert ((lse.double() - exact_lse).abs() <= lse_slack).all()


@pytest.mark.parametrize("bad", ["a query", "an early key", "an early value", "a channel", "values here and there"])
@pytest.mark.parametrize("dim", [64, 128])
def test_visible_nan_takes_no_longer(bad, dim):
    """A long prompt that has met a NaN is wrong, and not slow: ten times a clean one's time at most."""
    s = problem(65, [4096], heads=4, kv_heads=2, dim=dim, causal=True)
    starts, lengths, out = ints(s["starts"]), ints(s["lengths"]), torch.empty_like(s["q"])

    def best():
        times = []
        for _ in range(6):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            attention.attend(s["q"], s["k"], s["v"], out, starts, lengths, causal=True)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    clean = best()
    if bad == "a query":
        s["q"][50:60, 1] = math.nan
    elif bad == "an early key":
        s["k"][50, 0] = math.inf
    elif bad == "an early value":
        s["v"][50, :, 7] = math.inf
    elif bad == "a channel":
        s["v"][:, 1, 9] = math.nan
    else:
        s["v"][torch.rand(s["v"].shape, generator=generator(66), device="cuda") < 1e-4] = math.nan
    spent = best()
    want, _, slack, _ = define(s)
    assert torch.equal(~out.isfinite(), want.isnan())
    fine = ~want.isnan()
    assert (out.double() - want)[fine].abs().sub(slack[fine]).max() <= 0
    assert spent <= 10 * clean, (spent, clean)


@pytest.mark.parametrize("queries,keys,dim", [([1] * 40, [3000] * 40, 128), ([1] * 40, [200] * 40, 64), ([700, 300], None, 128), ([20, 1], [9000, 130], 64)])
def test_the_same_hundreds_of_times(queries, keys, dim):
    """Roles of a CTA that meet in another order each time."""
    s = problem(69, queries, keys, heads=8, kv_heads=2, dim=dim, causal=True)
    want, want_lse = check(s)
    k = {} if keys is None else {"k_starts": ints(s["k_starts"]), "k_lengths": ints(s["k_lengths"])}
    starts, lengths, out, lse = ints(s["starts"]), ints(s["lengths"]), torch.empty_like(want), torch.empty_like(want_lse)
    err, others = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(400):
        out.fill_(7.0)
        attention.attend(s["q"], s["k"], s["v"], out, starts, lengths, max_queries=max(queries), max_keys=max(keys or queries), causal=True, lse=lse, err=err, **k)
        others += (out != want).sum() + (lse != want_lse).sum()
    assert err.item() == 0 and others.item() == 0


@pytest.mark.parametrize("how", [dict(slopes=1e30), dict(slopes=2e38), dict(slopes=3.4e38), dict(cap=1e-30), dict(cap=1e-40), dict(cap=1e-45), dict(cap=3e38),
                                 dict(cap=1e30, scale=1e-10), dict(cap=1e-40, slopes=0.5), dict(cap=1e-40, distance_bias=3)])
@pytest.mark.parametrize("queries,keys", [([300], None), ([1, 3], [900, 200])])
def test_factors_at_the_ends_of_their_range(how, queries, keys):
    how = dict(how)
    if "slopes" in how:
        how["slopes"] = torch.full((4,), how["slopes"], device="cuda")
    if "distance_bias" in how:
        how = with_bias(how, 4)
    s = problem(67, queries, keys, heads=4, kv_heads=2, dim=64, causal=True, **how)
    s["q"][::3] = 0
    check(s)


@pytest.mark.parametrize("cap", [1e-46, 1e-60, 5e-324])
def test_a_cap_below_32_bits_is_a_cap(cap):
    check(problem(71, [300, 1], heads=4, kv_heads=2, dim=64, causal=True, cap=cap))


def test_a_scale_at_the_end_of_its_range():
    for value in (3e38, -3e38):
        s = problem(68, [300, 1], heads=4, kv_heads=2, dim=64, causal=True, scale=value)
        s["q"].zero_()
        check(s)


# -------------------------------------------------------------------------------- a layer

def layer_example():
    import importlib.util
    from pathlib import Path
    spec = importlib.util.spec_from_file_location("attention_layer", Path(__file__).resolve().parents[1] / "examples" / "attention_layer.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    return example


def test_the_layer_example_runs(capsys):
    seen = list(layer_example().main(6, 2, 64))
    assert [s[:2] for s in seen] == [("prompt", 500), ("token", 1), ("prompt", 1720), ("token", 4)]
    assert all(math.isfinite(s[2]) for s in seen) and capsys.readouterr().out.count("tokens") == 4


def test_the_layer_is_its_operators_one_after_the_other():
    """Prompts through the layer, bit for bit the operators' results, and tokens after them that see what the prompts left."""
    from laya_cuda import mx8
    example, g = layer_example(), generator(50)
    heads, kv, dim, prompts = 4, 2, 32, [40, 9]
    width, tokens = heads * dim, sum(prompts)
    weight, qkv, out = randn(g, width).float(), randn(g, (heads + 2 * kv) * dim, width).float() * 0.1, randn(g, width, width).float() * 0.1
    layer = example.AttentionLayer(weight, qkv, out, heads, kv)
    cache = example.Cache(2, 64, kv, dim, torch.bfloat16)
    x, r = randn(g, tokens, width).bfloat16(), randn(g, tokens, width).float()
    positions = torch.cat([torch.arange(n, device="cuda") for n in prompts])
    got = layer(x, r.clone(), ints([0, 40]), ints(prompts), positions, cache, 40)
    n8, total, projected = mx8.Matrix.empty(x, tokens, width), r.clone(), torch.empty(tokens, (heads + 2 * kv) * dim, dtype=torch.bfloat16, device="cuda")
    mx8.rms_norm(x, weight, n8, residual=total, sum_out=total)
    mx8.linear(n8, layer.qkv, projected)
    h = projected.view(tokens, heads + 2 * kv, dim)
    q, k = torch.empty_like(h[:, :heads]).contiguous(), torch.empty(tokens, kv, dim, dtype=torch.bfloat16, device="cuda")
    attention.rotary(h[:, :heads], positions, q, k=h[:, heads:-kv], k_out=k)
    rows = torch.cat([b * 64 + torch.arange(n, device="cuda") for b, n in enumerate(prompts)])
    assert torch.equal(cache.k[rows], k) and torch.equal(cache.v[rows], h[:, -kv:])
    attended = torch.empty_like(q)
    attention.attend(q, cache.k, cache.v, attended, ints([0, 40]), ints(prompts), cache.starts, ints(prompts), max_queries=40, max_keys=64, causal=True)
    a8 = mx8.Matrix.empty(x, tokens, width)
    mx8.quantize(attended.view(tokens, -1), a8)
    mx8.linear(a8, layer.out, total, residual=total)
    assert torch.equal(got, total)
    kept = cache.k[rows].clone()
    after = layer(x[:2], r[:2].clone(), ints([0, 1]), ints([1, 1]), torch.tensor(prompts, device="cuda"), cache, 1)
    assert torch.equal(cache.k[rows], kept) and cache.lengths.tolist() == [41, 10] and bool(after.isfinite().all())
