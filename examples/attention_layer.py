"""A pre-norm attention layer: projections in MX8, rotary positions and attention between them, a cache for single tokens.

    r += x;  n = rms_norm(r) * weight                       one kernel, n in MX8
    q, k, v = n W^T                                         one kernel, 16 bits
    q, k turned by their positions, in place                one kernel
    k, v into the cache                                     torch's indexing
    a = attention of q over the cache                       one kernel (the prompt's tokens, or one token for each sequence)
    r += a O^T                                              two kernels, a put into MX8 first

    python examples/attention_layer.py [heads] [kv_heads] [head_dim]

prints the layer's time and its distance from fp32 for prompts and for the tokens after them.
"""
import math
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "laya-cuda_b200"))

import torch  # noqa: E402

from laya_cuda import attention, mx8  # noqa: E402


class Cache:
    """Keys and values of `sequences` sequences with room for `room` tokens each; sequence b starts at row b * room."""

    def __init__(self, sequences, room, kv_heads, head_dim, dtype, device="cuda"):
        self.room = room
        self.k, self.v = (torch.empty(sequences * room, kv_heads, head_dim, dtype=dtype, device=device) for _ in range(2))
        self.starts = torch.arange(sequences, dtype=torch.int32, device=device) * room
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)


class AttentionLayer:
    """weight: fp32 [width]; qkv: [(heads + 2 kv_heads) head_dim][width]; out: [width][heads head_dim]."""

    def __init__(self, weight, qkv, out, heads, kv_heads, cap=0.0, eps=1e-6):
        self.weight, self.heads, self.kv_heads, self.cap, self.eps = weight.float(), heads, kv_heads, cap, eps
        self.head_dim = qkv.shape[0] // (heads + 2 * kv_heads)
        self.qkv, self.out = (self.pack(w) for w in (qkv, out))

    @staticmethod
    def pack(w):
        m = mx8.Matrix.empty(w, *w.shape)
        mx8.quantize(w, m)
        return m

    def __call__(self, x, residual, starts, lengths, positions, cache, most):
        """Adds x and then the layer's output to `residual`, in place.  The packed tokens' keys and values go to the cache behind those
        that it holds: token t of sequence b to row cache.starts[b] + positions[t].  `most`: no sequence has more of the tokens."""
        tokens, width = x.shape
        n = mx8.Matrix.empty(x, tokens, width)
        projected = torch.empty(tokens, self.qkv.rows, dtype=torch.bfloat16, device=x.device)
        mx8.rms_norm(x, self.weight, n, residual=residual, sum_out=residual, eps=self.eps)
        mx8.linear(n, self.qkv, projected)
        heads = projected.view(tokens, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = heads[:, : self.heads], heads[:, self.heads: -self.kv_heads], heads[:, -self.kv_heads:]
        attention.rotary(q, positions, q, k=k, k_out=k)
        sequence = torch.repeat_interleave(torch.arange(len(lengths), device=x.device), lengths, output_size=tokens)
        rows = cache.starts[sequence] + positions
        cache.k[rows], cache.v[rows] = k, v
        cache.lengths += lengths
        attended = torch.empty(tokens, self.heads, self.head_dim, dtype=q.dtype, device=x.device)
        attention.attend(q, cache.k, cache.v, attended, starts, lengths, cache.starts, cache.lengths, max_queries=most, max_keys=cache.room,
                         causal=True, cap=self.cap)
        a = mx8.Matrix.empty(x, tokens, self.out.cols)
        mx8.quantize(attended.view(tokens, -1), a)
        mx8.linear(a, self.out, residual, residual=residual)
        return residual


def reference(weight, qkv, out, heads, kv_heads, x, residual, lengths, cap=0.0, eps=1e-6):
    """The same layer in fp32 over whole sequences."""
    r = residual.float() + x.float()
    n = r / torch.sqrt((r * r).mean(1, keepdim=True) + eps) * weight
    dim = qkv.shape[0] // (heads + 2 * kv_heads)
    done = []
    for part in (n @ qkv.T).view(len(x), -1, dim).split(lengths):
        angle = torch.arange(len(part), device=x.device)[:, None, None] * 10000.0 ** (-2 * torch.arange(dim // 2, device=x.device) / dim)
        a, b = part[:, :-kv_heads, : dim // 2], part[:, :-kv_heads, dim // 2:]
        turned = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)
        q, k = turned[:, :heads], turned[:, heads:].repeat_interleave(heads // kv_heads, 1)
        v = part[:, -kv_heads:].repeat_interleave(heads // kv_heads, 1)
        s = torch.einsum("nhd,mhd->hnm", q, k) / math.sqrt(dim)
        s = cap * torch.tanh(s / cap) if cap else s
        s = s.masked_fill(torch.ones_like(s[0], dtype=torch.bool).triu(1), -math.inf)
        done.append(torch.einsum("hnm,mhd->nhd", torch.softmax(s, -1), v).reshape(len(part), -1))
    return r + torch.cat(done) @ out.T


def main(heads=12, kv_heads=4, head_dim=64):
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    width = heads * head_dim
    weight = 1 + 0.1 * rand(width)
    qkv, out = rand((heads + 2 * kv_heads) * head_dim, width) / width ** 0.5, rand(width, heads * head_dim) / width ** 0.5
    layer = AttentionLayer(weight, qkv, out, heads, kv_heads, cap=30.0)
    for prompts in ([500], [1000, 77, 640, 3]):
        whole = [n + 1 for n in prompts]
        x, r = rand(sum(whole), width).bfloat16(), rand(sum(whole), width)
        want = reference(weight, qkv, out, heads, kv_heads, x, r, whole, cap=30.0) - (r + x.float())
        last = torch.tensor(whole, device="cuda").cumsum(0) - 1
        before = torch.ones(len(x), dtype=torch.bool, device="cuda").index_fill_(0, last, False)
        cache = Cache(len(prompts), max(whole), kv_heads, head_dim, torch.bfloat16)
        starts = ints([sum(prompts[:b]) for b in range(len(prompts))])
        positions = torch.cat([torch.arange(n, device="cuda") for n in prompts])
        steps = [("prompt", before, starts, ints(prompts), positions, max(prompts)),
                 ("token", ~before, ints(range(len(prompts))), ints([1] * len(prompts)), torch.tensor(prompts, device="cuda"), 1)]
        for name, some, at, lengths, where, most in steps:
            mine, rest = x[some], r[some]
            base, scratch, held = rest + mine.float(), rest.clone(), cache.lengths.clone()
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            for k in range(23):
                if k == 3:
                    start.record()
                layer(mine, scratch, at, lengths, where, cache, most)
                cache.lengths.copy_(held)
            end.record()
            end.synchronize()
            got = layer(mine, rest, at, lengths, where, cache, most) - base
            off = ((got - want[some]).norm() / want[some].norm()).item()
            print(f"{len(mine):6d} tokens of {len(prompts)} sequences ({name}): {start.elapsed_time(end) / 20 * 1e3:8.1f} us, update {off:.4f} off fp32")
            yield name, len(mine), off


if __name__ == "__main__":
    list(main(*map(int, sys.argv[1:])))
