"""Rotary positions and attention with caps, biases and masks, as they are measured: cases, inputs, plain forms and
exact values.

  rotary   the first `dims` values of each head turned in pairs by position * f_k, f_k = theta^(-2k / dims):
             (a, b) -> magnitude * (a cos - b sin, a sin + b cos)
           pairs (2k, 2k + 1) interleaved, (k, k + dims / 2) in the half layout; the rest of the head is copied.
           Scaled for long contexts: linear (f_k / factor), ntk (theta * factor^(dims / (dims - 2))) and parts
           (f_k (g + (1 - g) / factor), g = clamp((length f_k / 2 pi - low) / (high - low), 0, 1)).
           Backward is the transposed map, from a gradient of the result to one of the input.
  attend   packed sequences; query i of a sequence of n queries and m keys is at p = i + m - n, and
             s = scale q . k,  s = cap tanh(s / cap),  s += bias,  out = softmax(s) v over the visible keys
           bias: -slope |j - p| for each head, or a table [heads][2 reach + 1] by j - p, cut off at +-reach.
           Key j is visible where j < prefix, or where it is in the query's document and inside the causal mask
           and the window.  `lse` is the logarithm of the sum of exp(s).
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _rotary(name, tokens, heads, kv_heads, dim, dims, type, interleaved=False, scaling="none", far=0, pad=0, backward=False):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dims": dims,
            "type": type, "interleaved": interleaved, "scaling": scaling, "far": far, "pad": pad, "backward": backward}


def _attend(name, sequences, queries, keys, heads, kv_heads, dim, type, ragged=False, cap=0.0, bias="none", reach=0,
            causal=False, window=-1, prefix=0, document=0, lse=False):
    """`keys` 0: self-attention, the keys are the queries' own tokens; otherwise a cache with room for `keys` tokens of each
    sequence.  `document`: mean length of the documents that a sequence is cut into, 0 for none."""
    return {"name": name, "op": "attend", "sequences": sequences, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "type": type, "ragged": ragged, "cap": cap, "bias": bias, "reach": reach,
            "causal": causal, "window": window, "prefix": prefix, "document": document, "lse": lse}


def listed():
    return [
        # A single token's queries and keys between the projection and attention: launch latency is all there is.
        _rotary("rotary one token", 1, 12, 12, 64, 64, "bf16"),
        # A short ragged batch, part of the head turned, rows inside a wider projection's buffer.
        _rotary("rotary part interleaved", 333, 16, 4, 80, 32, "f16", interleaved=True, scaling="ntk", pad=24),
        # A packed batch of long contexts, far positions.
        _rotary("rotary long batch", 16384, 32, 8, 128, 128, "bf16", scaling="parts", far=900000),
        # Gradients of a batch's queries and keys in 32 bits.
        _rotary("rotary gradient", 9001, 16, 16, 96, 96, "f32", scaling="linear", backward=True),
        # One new token of one sequence over a short cache: latency.
        _attend("attend one token", 1, 1, 96, 12, 12, 64, "f16", cap=30.0, causal=True),
        # A batch of single tokens over long caches: the caches' bytes count.
        _attend("attend single tokens", 16, 1, 32768, 32, 8, 128, "bf16", ragged=True, bias="slopes", causal=True),
        # A few questions' tokens over a cached state; the logarithms are for joining the result with another piece's.
        _attend("attend questions on a cache", 3, 24, 4099, 16, 4, 128, "bf16", ragged=True, causal=True, lse=True),
        # One request: a state that every token sees and questions that see the state and themselves.
        _attend("attend one request", 1, 1000, 0, 12, 12, 64, "f16", bias="table", reach=128, prefix=600, document=80),
        # The encoder's packed batch with a learned bias by distance.
        _attend("attend packed batch", 64, 1024, 0, 12, 12, 64, "f16", ragged=True, bias="table", reach=128),
        # Ragged prompts in documents, a sliding window, capped scores, heads of an odd size.
        _attend("attend windowed documents", 5, 4097, 0, 15, 5, 96, "bf16", ragged=True, cap=50.0, causal=True, window=1023,
                document=1500),
        # Long packed documents of a decoder's prompt.
        _attend("attend documents", 1, 8192, 0, 32, 8, 128, "bf16", causal=True, document=600),
        # One long prompt, capped scores.
        _attend("attend long prompt", 1, 16384, 0, 16, 4, 128, "bf16", cap=50.0, causal=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7, 8])
        if heads > 64:
            continue
        if rng.random() < 0.35:
            dim = rng.choice([32, 40, 64, 80, 96, 128, 128, 256])
            case = _rotary("", _log(rng, 1, 32768), heads, kv_heads, dim, rng.choice([dim, dim, dim // 4 * 2]),
                           rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.5, rng.choice(["none", "linear", "ntk", "parts"]),
                           rng.choice([0, 0, _log(rng, 1000, 10000000)]), rng.choice([0, 0, 1, 8, 24]), rng.random() < 0.25)
            if case["tokens"] * (heads + kv_heads) * dim > 16384 * 40 * 128:
                continue
        else:
            form = rng.choice(["tokens", "chunk", "prompt", "prompt"])
            sequences = _log(rng, 1, 64)
            if form == "tokens":
                queries, keys = rng.choice([1, 1, 1, 2, 5]), _log(rng, 16, 131072)
            elif form == "chunk":
                queries, keys = _log(rng, 6, 700), _log(rng, 700, 32768)
            else:
                queries, keys = _log(rng, 16, 16384), 0
            bias = rng.choice(["none", "none", "slopes", "table"])
            longest = keys or queries
            case = _attend("", sequences, queries, keys, heads, kv_heads, rng.choice([32, 64, 64, 72, 80, 96, 128, 128]),
                           rng.choice(["bf16", "f16"]), rng.random() < 0.6, rng.choice([0.0, 0.0, 20.0, 50.0]), bias,
                           rng.choice([16, 128, 1000]) if bias == "table" else 0, rng.random() < 0.6,
                           rng.choice([-1, -1, _log(rng, 1, 4096)]),
                           _log(rng, 1, longest) if keys == 0 and rng.random() < 0.3 else 0,
                           _log(rng, 30, 3000) if keys == 0 and rng.random() < 0.3 else 0, rng.random() < 0.2)
            if (sequences * queries * longest * heads * case["dim"] > 16384 * 16384 * 16 * 128
                    or sequences * longest * kv_heads * case["dim"] > 16 * 32768 * 8 * 128):
                continue
        del case["name"]
        return case


# ------------------------------------------------------------------------------------------------ a case's lengths and masks


def _lengths(case):
    """Queries and keys of each sequence; a fixed function of the case."""
    rng = random.Random(case["sequences"] * 1000003 + case["queries"] * 1009 + case["keys"])
    n, most = case["sequences"], case["keys"] or case["queries"]
    longest = [most] + [rng.randint(max(1, most // 8), most) if case["ragged"] else most for _ in range(n - 1)]
    if not case["keys"]:
        return longest, longest
    return [min(case["queries"], m) for m in longest], longest


def _documents(case, length, which):
    """The document of each token of sequence `which`: runs of random length."""
    rng = random.Random(which * 7919 + length)
    out = []
    while len(out) < length:
        out += [len(out)] * max(1, int(rng.expovariate(1 / case["document"])))
    return out[:length]


def _sees(case, p, j, prefix, doc_p, doc_j):
    """Which keys are visible; p and doc_p broadcast against j and doc_j."""
    see = torch.ones_like(p + j, dtype=torch.bool)
    if case["causal"]:
        see = see & (j <= p)
    if case["window"] >= 0:
        see = see & (j >= p - case["window"])
        if not case["causal"]:
            see = see & (j <= p + case["window"])
    if doc_p is not None:
        see = see & (doc_p == doc_j)
    return see | (j < prefix)


# ------------------------------------------------------------------------------------------------ inputs


def _values(g, tokens, heads, dim, dtype, pad=0):
    """[tokens][heads][dim], a view of rows `pad` values wider."""
    store = torch.randn(tokens, heads * dim + pad, generator=g, device="cuda").to(dtype)
    return store[:, : heads * dim].view(tokens, heads, dim) if not pad else store[:, : heads * dim].unflatten(1, (heads, dim))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["op"] == "rotary":
        n = case["tokens"]
        s["q"], s["k"] = _values(g, n, heads, dim, dtype, case["pad"]), _values(g, n, kv, dim, dtype, case["pad"])
        s["positions"] = torch.arange(n, device="cuda") + case["far"] + int(torch.randint(0, 50, (1,), generator=g, device="cuda"))
        s["q_out"], s["k_out"] = (torch.zeros(n, h, dim, dtype=dtype, device="cuda") for h in (heads, kv))
        return s
    queries, keys = _lengths(case)
    device = {"device": "cuda", "dtype": torch.int32}
    s["host_queries"], s["host_keys"] = queries, keys
    s["lengths"], s["k_lengths"] = torch.tensor(queries, **device), torch.tensor(keys, **device)
    s["starts"] = torch.tensor([sum(queries[:b]) for b in range(len(queries))], **device)
    if case["keys"]:
        s["q"] = _values(g, sum(queries), heads, dim, dtype)
        s["k"], s["v"] = (_values(g, len(keys) * case["keys"], kv, dim, dtype) for _ in range(2))
        s["k_starts"] = torch.arange(len(keys), **device) * case["keys"]
    else:  # slices of one projection's result
        packed = _values(g, sum(queries), heads + 2 * kv, dim, dtype)
        s["q"], s["k"], s["v"] = packed[:, :heads], packed[:, heads: heads + kv], packed[:, heads + kv:]
        s["k_starts"] = s["starts"]
    for t in (s["q"], s["k"]):  # a few channels larger than the others
        t *= torch.exp(0.4 * torch.randn(dim, generator=g, device="cuda")).to(dtype)
    s["out"] = torch.zeros(sum(queries), heads, dim, dtype=dtype, device="cuda")
    s["lse"] = torch.zeros(sum(queries), heads, device="cuda") if case["lse"] else None
    s["scale"] = 1 / math.sqrt(dim)
    s["slopes"] = s["table"] = s["prefix"] = s["documents"] = None
    if case["bias"] == "slopes":
        s["slopes"] = torch.exp2(-8 * torch.arange(1, heads + 1, device="cuda") / heads)
    if case["bias"] == "table":
        s["table"] = 0.7 * torch.randn(heads, 2 * case["reach"] + 1, generator=g, device="cuda")
    if case["prefix"]:
        s["prefix"] = torch.tensor([max(1, n * case["prefix"] // case["queries"]) for n in keys], **device)
    if case["document"]:
        s["documents"] = torch.tensor([d for b, n in enumerate(keys) for d in _documents(case, n, b)], **device)
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _frequencies(case):
    """f_k in 64 bits."""
    theta, dims = 10000.0, case["dims"]
    if case["scaling"] == "ntk":
        theta *= 8.0 ** (dims / (dims - 2))
    f = theta ** (-torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / dims)
    if case["scaling"] == "linear":
        f = f / 8.0
    if case["scaling"] == "parts":
        keep = ((4096 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        f = f * (keep + (1 - keep) / 8.0)
    return f


def _magnitude(case):
    return 0.1 * math.log(8.0) + 1 if case["scaling"] == "parts" else 1.0


def _turn(case, x, cos, sin):
    dims = case["dims"]
    y = x.float()
    a, b = (y[..., 0:dims:2], y[..., 1:dims:2]) if case["interleaved"] else (y[..., : dims // 2], y[..., dims // 2: dims])
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.stack(turned, -1).flatten(-2) if case["interleaved"] else torch.cat(turned, -1)
    return torch.cat([turned, y[..., dims:]], -1).to(x.dtype)


def _plain_attend(s, heads, first, last):
    """Sequences first .. last, some of the kv heads, as one padded batch."""
    case = s["case"]
    kv = heads.stop - heads.start
    group, dim = case["heads"] // case["kv_heads"], case["dim"]
    n, m = max(s["host_queries"][first:last]), max(s["host_keys"][first:last])
    i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    nq, nk = s["lengths"][first:last, None], s["k_lengths"][first:last, None]
    at_q = (s["starts"][first:last, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    at_k = (s["k_starts"][first:last, None] + j).clamp(max=s["k"].shape[0] - 1).long()
    q = s["q"][:, heads.start * group: heads.stop * group][at_q].float()  # [batch][n][heads][dim]
    k, v = (s[name][:, heads][at_k].float().transpose(1, 2) for name in ("k", "v"))
    q = q.view(-1, n, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(-1, kv, group * n, dim)
    x = (q @ k.transpose(2, 3)).view(-1, kv, group, n, m)
    x *= s["scale"]
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    p = (i + nk - nq)[:, :, None]  # [batch][n][1]
    distance = j - p
    if s["slopes"] is not None:
        x -= s["slopes"][heads.start * group: heads.stop * group].view(kv, group, 1, 1) * distance.abs()[:, None, None]
    if s["table"] is not None:
        table = s["table"][heads.start * group: heads.stop * group]
        by_distance = distance.clamp(-case["reach"], case["reach"]) + case["reach"]
        x += table[:, by_distance].view(kv, group, -1, n, m).permute(2, 0, 1, 3, 4)
    prefix = s["prefix"][first:last, None, None] if s["prefix"] is not None else 0
    doc = s["documents"]
    see = _sees(case, p, j, prefix, None if doc is None else doc[at_q][:, :, None], None if doc is None else doc[at_k][:, None])
    see = see & (j < nk[:, :, None])
    x.masked_fill_(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = x.sum(-1, keepdim=True)
    v = torch.where((j < nk)[:, None, :, None], v, torch.zeros_like(v))
    y = (x.view(-1, kv, group * n, m) @ v).view(-1, kv, group, n, dim) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total)).squeeze(-1)
    real = i < nq
    y = y.permute(0, 3, 1, 2, 4).reshape(-1, n, kv * group, dim)[real]
    return y.to(s["out"].dtype), lse.permute(0, 3, 1, 2).reshape(-1, n, kv * group)[real]


def _run_plain(s):
    case = s["case"]
    if case["op"] == "rotary":
        angle = s["positions"].double()[:, None] * _frequencies(case)
        cos, sin = (_magnitude(case) * t.float()[:, None] for t in (torch.cos(angle), torch.sin(angle)))
        if case["backward"]:
            sin = -sin
        return {"q": _turn(case, s["q"], cos, sin), "k": _turn(case, s["k"], cos, sin)}
    # At most 2^29 scores at a time: all sequences that fit, or some heads of one.
    n, m = max(s["host_queries"]), max(s["host_keys"])
    group = case["heads"] // case["kv_heads"]
    batch = max(1, min(case["sequences"], (1 << 29) // (n * m * case["heads"])))
    some = case["kv_heads"] if batch > 1 else max(1, min(case["kv_heads"], (1 << 29) // (n * m * group)))
    parts = []
    for first in range(0, case["sequences"], batch):
        row = [_plain_attend(s, slice(h, min(h + some, case["kv_heads"])), first, min(first + batch, case["sequences"]))
               for h in range(0, case["kv_heads"], some)]
        parts.append([torch.cat(t, 1) for t in zip(*row)])
    out, lse = (torch.cat(t) for t in zip(*parts))
    return {"out": out, "lse": lse} if case["lse"] else out


# ------------------------------------------------------------------------------------------------ one pass


def _package():
    where = os.path.join(os.getcwd(), "laya-cuda_b200")
    if where not in sys.path:
        sys.path.insert(0, where)
    from laya_cuda import attention
    return attention


def _run_own(s):
    attention = sys.modules.get("laya_cuda.attention") or _package()
    case = s["case"]
    if case["op"] == "rotary":
        attention.rotary(s["q"], s["positions"], s["q_out"], k=s["k"], k_out=s["k_out"], dims=case["dims"],
                         interleaved=case["interleaved"], scaling=case["scaling"],
                         factor=1.0 if case["scaling"] == "none" else 8.0, length=4096, low=1.0, high=32.0,
                         magnitude=_magnitude(case), backward=case["backward"])
        return {"q": s["q_out"], "k": s["k_out"]}
    window = case["window"]
    attention.attend(s["q"], s["k"], s["v"], s["out"], s["starts"], s["lengths"], k_starts=s["k_starts"], k_lengths=s["k_lengths"],
                     max_queries=max(s["host_queries"]), max_keys=max(s["host_keys"]), scale=s["scale"], cap=case["cap"],
                     causal=case["causal"], window=(window, -1 if case["causal"] else window), prefix=s["prefix"],
                     documents=s["documents"], slopes=s["slopes"], distance_bias=s["table"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]} if case["lse"] else s["out"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    heads, kv, dim, size = case["heads"], case["kv_heads"], case["dim"], SIZE[case["type"]]
    if case["op"] == "rotary":
        return {"bytes": case["tokens"] * (2 * (heads + kv) * dim * size + 8), "flops": 3 * case["tokens"] * (heads + kv) * case["dims"]}
    queries, keys = _lengths(case)
    pairs = read = 0
    for b, (n, m) in enumerate(zip(queries, keys)):
        p, j = torch.arange(m - n, m)[:, None], torch.arange(m)
        prefix = max(1, m * case["prefix"] // case["queries"]) if case["prefix"] else 0
        if case["document"] or (prefix and (case["causal"] or case["window"] >= 0)):
            doc = torch.tensor(_documents(case, m, b)) if case["document"] else torch.zeros(m, dtype=torch.long)
            for at in range(0, n, 1024):
                pairs += int(_sees(case, p[at: at + 1024], j, prefix, doc[p[at: at + 1024]], doc).sum())
            read += m
        else:
            low = (p - case["window"]).clamp(min=0) if case["window"] >= 0 else torch.zeros_like(p)
            high = p if case["causal"] else (p + case["window"]).clamp(max=m - 1) if case["window"] >= 0 else torch.full_like(p, m - 1)
            pairs += int((high - low + 1).sum())
            read += int(high.max() - low.min() + 1)
    moved = sum(queries) * heads * (2 * dim * size + (4 if case["lse"] else 0)) + 2 * read * kv * dim * size
    if case["bias"] == "table":
        moved += 4 * heads * (2 * case["reach"] + 1)
    return {"bytes": moved, "flops": 4 * pairs * heads * dim}


# ------------------------------------------------------------------------------------------------ exact values
#
# In 64 bits, from the definitions, one sequence and head at a time.


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        dims, k = case["dims"], torch.arange(case["dims"] // 2, device="cuda")
        step = torch.exp(-2.0 * k.double() / dims * math.log(10000.0))
        if case["scaling"] == "ntk":
            step = step * torch.exp(-2.0 * k.double() / (dims - 2) * math.log(8.0))
        if case["scaling"] == "linear":
            step = step * 0.125
        if case["scaling"] == "parts":
            turns = 4096 / (2 * math.pi / step)
            step = torch.where(turns >= 32, step, torch.where(turns <= 1, step / 8, step * (1 + 7 * (turns - 1) / 31) / 8))
        first, second = (2 * k, 2 * k + 1) if case["interleaved"] else (k, k + dims // 2)
        phase = torch.polar(torch.full_like(step, _magnitude(case)).expand(case["tokens"], -1),
                            s["positions"].double()[:, None] * step * (-1 if case["backward"] else 1))[:, None]
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            turned = torch.complex(x[..., first], x[..., second]) * phase
            x[..., first], x[..., second] = turned.real, turned.imag
            out[name] = x
        return out
    if sum(n * m for n, m in zip(s["host_queries"], s["host_keys"])) * case["heads"] > 1 << 33:
        return None
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["out"].shape[:2], dtype=torch.float64, device="cuda")
    q_at = k_at = 0
    for b, (n, m) in enumerate(zip(s["host_queries"], s["host_keys"])):
        p, j = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")
        doc = s["documents"][k_at: k_at + m] if case["document"] else None
        hidden = ~_sees(case, p, j, max(1, m * case["prefix"] // case["queries"]) if case["prefix"] else 0,
                        None if doc is None else doc[p], doc)
        for h in range(case["heads"]):
            q = s["q"][q_at: q_at + n, h].double()
            k, v = (s[name][k_at: k_at + m, h // group].double() for name in ("k", "v"))
            x = torch.mm(q, k.t()) / math.sqrt(case["dim"])
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            if case["bias"] == "slopes":
                x = x - (p - j).abs() * s["slopes"][h].double()
            if case["bias"] == "table":
                x = x + s["table"][h].double()[(j - p + case["reach"]).clamp(0, 2 * case["reach"])]
            x[hidden] = -math.inf
            lse[q_at: q_at + n, h] = torch.logsumexp(x, 1)
            out[q_at: q_at + n, h] = torch.mm(torch.softmax(x, 1), v)
        q_at, k_at = q_at + n, k_at + (case["keys"] or m)
    return {"out": out, "lse": lse} if case["lse"] else out
