"""The 8-bit linear layer's operators, as they are measured: cases, inputs, plain forms and exact values.

Four operators work on the MX8 format: E4M3 values in rows, with one power-of-two scale (E8M0) for each block of 32
consecutive values of a row.

  quantize     a matrix in 16 or 32 bits into MX8 (weights once, activations where no other kernel writes them)
  dequantize   an MX8 matrix back into 16 or 32 bits
  rms_norm     h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, y written in MX8 and h for the next layer
  linear       act(X W^T + bias) + residual, or act(X G^T + bias_g) * (X W^T + bias) + residual, from MX8 operands,
               written in 16 bits or in MX8 for the next product

A block's scale is 2^e with e = floor(log2 a) - 8, and one more where a / 2^floor(log2 a) > 1.75, a the block's largest
magnitude: the smallest power of two under which no value passes 448, E4M3's largest.

Scales are stored in tiles of 128 rows x 4 blocks, 512 bytes each, tile (row / 128, block / 4) row-major; inside a
tile the scale of (row, block) is byte (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "none": 0}


def listed():
    return [
        # One token's activations before a projection: launch latency is all there is.
        {"name": "quantize one token", "op": "quantize", "rows": 1, "cols": 768, "pitch": 768, "type": "bf16"},
        # A projection's fp32 checkpoint weights, put into 8 bits at load.
        {"name": "quantize weights", "op": "quantize", "rows": 9216, "cols": 4096, "pitch": 4096, "type": "f32"},
        # A short packed batch of odd width, read back (a head that works in 16 bits).
        {"name": "dequantize ragged", "op": "dequantize", "rows": 77, "cols": 1000, "pitch": 1003, "type": "f16"},
        # A large packed batch of activations, read back.
        {"name": "dequantize batch", "op": "dequantize", "rows": 16384, "cols": 4096, "pitch": 4096, "type": "bf16"},
        # The norm of one token between two products, the residual stream in 32 bits as the encoder keeps it.
        {"name": "norm one token", "op": "rms_norm", "rows": 1, "cols": 4096, "pitch": 4096, "type": "bf16", "sum": "f32"},
        # A ragged batch of a narrow model whose rows are slices of a wider buffer.
        {"name": "norm ragged", "op": "rms_norm", "rows": 333, "cols": 1000, "pitch": 1012, "type": "f16", "sum": "f16"},
        # A full packed batch, bf16 throughout.
        {"name": "norm batch", "op": "rms_norm", "rows": 16384, "cols": 4096, "pitch": 4096, "type": "bf16", "sum": "bf16"},
        # A single token through an output projection onto the residual stream: the weights' bytes count.
        {"name": "linear one token", "op": "linear", "rows": 1, "cols": 4096, "features": 4096, "type": "bf16",
         "activation": "none", "gated": False, "bias": True, "residual": "f32"},
        # A few questions' tokens through a gated up-projection of odd width, in 8 bits for the next product.
        {"name": "linear few tokens gated", "op": "linear", "rows": 24, "cols": 2048, "features": 5461, "type": "mx8",
         "activation": "silu", "gated": True, "bias": False, "residual": "none"},
        # One request of the encoder's width: bias and exact-erf GELU, ragged depth.
        {"name": "linear one request", "op": "linear", "rows": 511, "cols": 776, "features": 2304, "type": "f16",
         "activation": "gelu", "gated": False, "bias": True, "residual": "none"},
        # A packed batch through the gated up-projection.
        {"name": "linear batch gated", "op": "linear", "rows": 8192, "cols": 2048, "features": 5632, "type": "mx8",
         "activation": "silu", "gated": True, "bias": False, "residual": "none"},
        # A large packed batch through a square projection with the residual's addition.
        {"name": "linear batch residual", "op": "linear", "rows": 16384, "cols": 4096, "features": 4096, "type": "bf16",
         "activation": "none", "gated": False, "bias": False, "residual": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "dequantize", "rms_norm", "linear", "linear", "linear"])
    while True:
        if op == "linear":
            case = {"op": op, "rows": _log(rng, 1, 16384), "cols": _log(rng, 32, 8192), "features": _log(rng, 32, 8192),
                    "type": rng.choice(["bf16", "f16", "mx8"]), "activation": rng.choice(["none", "relu", "gelu", "silu"]),
                    "gated": rng.random() < 0.4, "bias": rng.random() < 0.5,
                    "residual": rng.choice(["none", "bf16", "f16", "f32"])}
            if case["gated"] and case["activation"] in ("none", "relu"):
                case["activation"] = "silu"
            if rng.random() < 0.7:  # most models' sizes are multiples of 64
                for k in ("cols", "features"):
                    case[k] = max(64, case[k] // 64 * 64)
            if case["rows"] * case["cols"] * case["features"] * (2 if case["gated"] else 1) <= 16384 * 4096 * 4096:
                return case
        else:
            cols = _log(rng, 32, 16384)
            if rng.random() < 0.7:
                cols = max(32, cols // 32 * 32)
            case = {"op": op, "rows": _log(rng, 1, 32768), "cols": cols, "pitch": cols + rng.choice([0, 0, 0, 1, 8, 64]),
                    "type": rng.choice(["bf16", "f16", "f32"])}
            if op == "rms_norm":
                case["sum"] = rng.choice([case["type"], "f32"])
            if case["rows"] * case["cols"] <= 9216 * 4096:
                return case


# ------------------------------------------------------------------------------------------------ the format, plainly


def _up(n, m):
    return -(-n // m) * m


def _tiles(scales, rows, blocks):
    """[rows][blocks] scale bytes -> the tiled store; bytes outside the matrix are 0."""
    full = torch.zeros(_up(rows, 128), _up(blocks, 4), dtype=torch.uint8, device=scales.device)
    full[:rows, :blocks] = scales
    return full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _untile(tiles, rows, blocks):
    k = _up(blocks, 4) // 4
    return tiles.view(-1, k, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, 4 * k)[:rows, :blocks]


def _blocks(v):
    """fp32 [rows][cols] -> [rows][blocks][32], zeros past the last column."""
    rows, cols = v.shape
    if cols % 32:
        v = torch.cat([v, v.new_zeros(rows, _up(cols, 32) - cols)], 1)
    return v.reshape(rows, -1, 32)


def _quantize(v):
    """fp32 [rows][cols] -> E4M3 values [rows][pitch] (pitch: cols up to a multiple of 16, zeros there) and tiled scales."""
    rows, cols = v.shape
    b = _blocks(v)
    bits = b.abs().amax(-1).view(torch.int32)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=0)
    inverse = ((254 - byte) << 23).view(torch.float32)
    q = (b * inverse[..., None]).to(torch.float8_e4m3fn).view(torch.uint8).reshape(rows, -1)[:, : _up(cols, 16)]
    return q.contiguous(), _tiles(byte.to(torch.uint8), rows, b.shape[1])


def _dequantize(q, tiles, cols):
    rows = q.shape[0]
    blocks = _up(cols, 32) // 32
    scale = _untile(tiles, rows, blocks).view(torch.float8_e8m0fnu).to(torch.float32)
    return (_blocks(q[:, :cols].view(torch.float8_e4m3fn).to(torch.float32)) * scale[..., None]).reshape(rows, -1)[:, :cols]


# ------------------------------------------------------------------------------------------------ inputs


def _activations(g, rows, cols, pitch, dtype):
    """Rows as a layer sees them: a few channels much larger than the others.  A view of a buffer `pitch` wide."""
    channel = torch.exp(0.8 * torch.randn(cols, generator=g, device="cuda"))
    store = torch.zeros(rows, pitch, dtype=dtype, device="cuda")
    store[:, :cols] = torch.randn(rows, cols, generator=g, device="cuda") * channel
    return store[:, :cols]


def _weight(g, rows, cols):
    return torch.randn(rows, cols, generator=g, device="cuda") / math.sqrt(cols)


def _empty_mx8(rows, cols):
    q = torch.zeros(rows, _up(cols, 16), dtype=torch.uint8, device="cuda")
    return q, torch.zeros(_up(rows, 128) * _up(cols, 128) // 32, dtype=torch.uint8, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, cols = case["op"], case["rows"], case["cols"]
    s = {"case": case}
    if op == "linear":
        n = case["features"]
        s["x"] = _quantize(_activations(g, rows, cols, cols, torch.float32))
        s["w"] = _quantize(_weight(g, n, cols))
        s["gate"] = _quantize(_weight(g, n, cols)) if case["gated"] else None
        s["bias"] = 0.1 * torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s["gate_bias"] = 0.1 * torch.randn(n, generator=g, device="cuda") if case["bias"] and case["gated"] else None
        s["residual"] = None
        if case["residual"] != "none":
            s["residual"] = torch.randn(rows, n, generator=g, device="cuda").to(TYPES[case["residual"]])
        s["out"] = _empty_mx8(rows, n) if case["type"] == "mx8" else torch.zeros(rows, n, dtype=TYPES[case["type"]], device="cuda")
    elif op == "dequantize":
        s["x"] = _quantize(_activations(g, rows, cols, cols, torch.float32))
        s["out"] = torch.zeros(rows, case["pitch"], dtype=TYPES[case["type"]], device="cuda")[:, :cols]
    else:
        s["x"] = _activations(g, rows, cols, case["pitch"], TYPES[case["type"]])
        s["out"] = _empty_mx8(rows, cols)
        if op == "rms_norm":
            s["weight"] = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
            s["residual"] = torch.randn(rows, cols, generator=g, device="cuda").to(TYPES[case["sum"]])
            s["sum"] = torch.zeros(rows, cols, dtype=TYPES[case["sum"]], device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ one pass


def _values(mx8):
    """An MX8 matrix as the 8-bit numbers that it holds."""
    q, scales = mx8
    return {"values": q.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


def _act(v, name):
    if name == "relu":
        return torch.clamp(v, min=0)
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "quantize":
        return _values(_quantize(s["x"].float()))
    if op == "dequantize":
        return _dequantize(*s["x"], case["cols"]).to(TYPES[case["type"]])
    if op == "rms_norm":
        h = s["x"].float() + s["residual"].float()
        y = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"]
        return {"sum": h.to(TYPES[case["sum"]]), **_values(_quantize(y))}
    x = _dequantize(*s["x"], case["cols"])
    y = x @ _dequantize(*s["w"], case["cols"]).T
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["gate"] is not None:
        v = x @ _dequantize(*s["gate"], case["cols"]).T
        if s["gate_bias"] is not None:
            v = v + s["gate_bias"]
        y = _act(v, case["activation"]) * y
    else:
        y = _act(y, case["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return _values(_quantize(y)) if case["type"] == "mx8" else y.to(TYPES[case["type"]])


def _package():
    where = os.path.join(os.getcwd(), "laya-cuda_b200")
    if where not in sys.path:
        sys.path.insert(0, where)
    from laya_cuda import mx8
    return mx8


def _run_own(s):
    mx8 = sys.modules.get("laya_cuda.mx8") or _package()
    case, op = s["case"], s["case"]["op"]
    rows, cols = case["rows"], case["cols"]
    if op == "quantize":
        mx8.quantize(s["x"], mx8.Matrix(*s["out"], rows, cols))
        return _values(s["out"])
    if op == "dequantize":
        mx8.dequantize(mx8.Matrix(*s["x"], rows, cols), s["out"])
        return s["out"]
    if op == "rms_norm":
        mx8.rms_norm(s["x"], s["weight"], mx8.Matrix(*s["out"], rows, cols), residual=s["residual"], sum_out=s["sum"], eps=EPS)
        return {"sum": s["sum"], **_values(s["out"])}
    n = case["features"]
    mx8.linear(mx8.Matrix(*s["x"], rows, cols), mx8.Matrix(*s["w"], n, cols),
               mx8.Matrix(*s["out"], rows, n) if case["type"] == "mx8" else s["out"], bias=s["bias"],
               gate=mx8.Matrix(*s["gate"], n, cols) if case["gated"] else None, gate_bias=s["gate_bias"],
               activation=case["activation"], residual=s["residual"])
    return _values(s["out"]) if case["type"] == "mx8" else s["out"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    op, rows, cols = case["op"], case["rows"], case["cols"]
    mx8 = lambda r, c: r * c + r * -(-c // 32)  # noqa: E731
    if op == "linear":
        n, weights = case["features"], 2 if case["gated"] else 1
        out = mx8(rows, n) if case["type"] == "mx8" else rows * n * SIZE[case["type"]]
        vectors = 4 * n * weights if case["bias"] else 0
        return {"bytes": mx8(rows, cols) + weights * mx8(n, cols) + out + rows * n * SIZE[case["residual"]] + vectors,
                "flops": 2 * rows * cols * n * weights}
    size = rows * cols * SIZE[case["type"]]
    if op == "rms_norm":
        return {"bytes": size + 2 * rows * cols * SIZE[case["sum"]] + 4 * cols + mx8(rows, cols), "flops": 8 * rows * cols}
    return {"bytes": size + mx8(rows, cols), "flops": 2 * rows * cols}


# ------------------------------------------------------------------------------------------------ exact values
#
# In 64 bits, from the definitions.  The exact value of a number that is written in 16 or 8 bits is the number before
# that rounding (for an E4M3 value, the result over its block's scale).  The scales of computed results have none:
# a comparison decides them, and they are powers of two.


def _exact_mx8(q, tiles, cols):
    row = torch.arange(q.shape[0], device="cuda")[:, None]
    block = (torch.arange(cols, device="cuda") // 32)[None, :]
    per_row = -(-cols // 128)
    at = (row // 128 * per_row + block // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + block % 4
    byte = q[:, :cols].long()
    power, fraction = byte // 8 % 16, byte % 8
    v = torch.where(power > 0, torch.ldexp(1 + fraction.double() / 8, power - 7), torch.ldexp(fraction.double() / 8, torch.full_like(power, -6)))
    return torch.where(byte > 127, -v, v) * torch.exp2(tiles[at.reshape(-1)].view(at.shape).double() - 127)


def _exact_values(y, want_scales):
    """What an MX8 matrix stands for, over its scales, and the scales where they are wanted."""
    rows, cols = y.shape
    wide, per_row = -(-cols // 32), -(-cols // 128)
    padded = torch.zeros(rows, wide * 32, dtype=torch.float64, device="cuda")
    padded[:, :cols] = y
    largest = padded.abs().reshape(rows, wide, 32).max(2).values
    mantissa, power = torch.frexp(largest)  # largest = mantissa * 2^power, mantissa in [0.5, 1)
    e = (power - 9 + (mantissa > 0.875)).double().clamp(min=-127)
    e = torch.where(largest > 0, e, torch.full_like(e, -127))
    values = (padded.reshape(rows, wide, 32) / torch.exp2(e)[:, :, None]).reshape(rows, -1)[:, : -(-cols // 16) * 16]
    if not want_scales:
        return {"values": values, "scales": None}
    store = torch.full((-(-rows // 128) * per_row * 512,), 2.0 ** -127, dtype=torch.float64, device="cuda")
    row, block = torch.arange(rows, device="cuda")[:, None], torch.arange(wide, device="cuda")[None, :]
    store[(row // 128 * per_row + block // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + block % 4] = torch.exp2(e)
    return {"values": values, "scales": store}


def exact(case, seed):
    s = prepare(case, seed)
    op, cols = case["op"], case["cols"]
    if op == "quantize":
        return _exact_values(s["x"].double(), True)
    if op == "dequantize":
        return _exact_mx8(*s["x"], cols)
    if op == "rms_norm":
        total = s["x"].double() + s["residual"].double()
        norm = torch.linalg.vector_norm(total, dim=1, keepdim=True)
        y = s["weight"].double() * total * torch.rsqrt(norm ** 2 / cols + EPS)
        return {"sum": total, **_exact_values(y, False)}
    x = _exact_mx8(*s["x"], cols)
    y = torch.mm(x, _exact_mx8(*s["w"], cols).t())
    if case["bias"]:
        y += s["bias"].double()
    name = case["activation"]
    at = y
    if case["gated"]:
        at = torch.mm(x, _exact_mx8(*s["gate"], cols).t())
        if case["bias"]:
            at += s["gate_bias"].double()
    if name == "relu":
        at = torch.where(at > 0, at, torch.zeros_like(at))
    elif name == "gelu":
        at = at * 0.5 * torch.erfc(-at / math.sqrt(2))
    elif name == "silu":
        at = at * torch.sigmoid(at)
    y = at * y if case["gated"] else at
    if case["residual"] != "none":
        y = y + s["residual"].double()
    return _exact_values(y, False) if case["type"] == "mx8" else y
