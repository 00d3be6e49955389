"""A pre-norm gated feed-forward block in MX8: the weights put into 8 bits once, then, for each batch of
packed tokens,

    r += x;  n = rms_norm(r) * weight        one kernel, n in MX8
    a = silu(n G^T) * (n U^T)                one kernel, a in MX8
    r += a D^T                               one kernel

    python examples/mx8_feed_forward.py [width] [hidden]

prints the block's time and its distance from fp32 for one token and for packed batches.
"""
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "laya-cuda_b200"))

import torch  # noqa: E402

from laya_cuda import mx8  # noqa: E402


class FeedForward:
    """weight: fp32 [width]; gate, up: [hidden][width]; down: [width][hidden]."""

    def __init__(self, weight, gate, up, down, eps=1e-6):
        self.weight, self.eps = weight.float(), eps
        self.gate, self.up, self.down = (self.pack(w) for w in (gate, up, down))

    @staticmethod
    def pack(w):
        m = mx8.Matrix.empty(w, *w.shape)
        mx8.quantize(w, m, stream=torch.cuda.current_stream().cuda_stream)
        return m

    def buffers(self, tokens, like):
        """What a batch of up to this many tokens needs beside the residual stream; reuse it."""
        return (mx8.Matrix.empty(like, tokens, self.up.cols), mx8.Matrix.empty(like, tokens, self.up.rows))

    @staticmethod
    def first(m, rows):
        """The first rows of a matrix (tiles of scales follow one another by rows, so they start at the same byte)."""
        return m if m.rows == rows else mx8.Matrix(m.values[:rows], m.scales, rows, m.cols)

    def __call__(self, x, residual, buffers):
        """Adds x and then the block's output to `residual`, in place."""
        normed, hidden = (self.first(m, x.shape[0]) for m in buffers)
        stream = torch.cuda.current_stream().cuda_stream
        mx8.rms_norm(x, self.weight, normed, residual=residual, sum_out=residual, eps=self.eps, stream=stream)
        mx8.linear(normed, self.up, hidden, gate=self.gate, activation="silu", stream=stream)
        mx8.linear(hidden, self.down, residual, residual=residual, stream=stream)
        return residual


def reference(weight, gate, up, down, x, residual, eps=1e-6):
    """The same block in fp32."""
    r = residual.float() + x.float()
    n = r / torch.sqrt((r * r).mean(1, keepdim=True) + eps) * weight
    return r + (torch.nn.functional.silu(n @ gate.T) * (n @ up.T)) @ down.T


def main(width=768, hidden=2048):
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    weight = 1 + 0.1 * rand(width)
    gate, up, down = rand(hidden, width) / width ** 0.5, rand(hidden, width) / width ** 0.5, rand(width, hidden) / hidden ** 0.5
    block = FeedForward(weight, gate, up, down)
    for tokens in (1, 512, 16384):
        x, r = rand(tokens, width).bfloat16(), rand(tokens, width)
        buffers = block.buffers(tokens, x)
        want = reference(weight, gate, up, down, x, r)
        base = r + x.float()
        off = ((block(x, r.clone(), buffers) - want).norm() / (want - base).norm()).item()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            block(x, r, buffers)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        for k in range(23):
            if k == 3:
                start.record()
            graph.replay()
        end.record()
        end.synchronize()
        print(f"{tokens:6d} tokens: {start.elapsed_time(end) / 20 * 1e3:8.1f} us, update {off:.4f} off fp32")
        yield tokens, off


if __name__ == "__main__":
    list(main(*map(int, sys.argv[1:])))
