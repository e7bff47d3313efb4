"""One attention layer serving several requests on a GPU: their prompts are written to a paged cache, then every step brings
one new token of each, which is normalised, rotated, written and attended with.

    python examples/attention_serving.py [--requests 16] [--prompt 1000] [--steps 32] [--cache bfloat16|int8|float8_e4m3fn]

The projections are torch products with random weights.  The last step is checked against attention computed from the values
that the cache holds, in 64 bits, and the time of a step (a captured CUDA graph) is printed.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from lapis_b200 import attention  # noqa: E402


class Layer:
    """Weights of the layer and the tables of its rotation."""

    def __init__(self, width, q_heads, kv_heads, dim, places, device):
        self.q_heads, self.kv_heads, self.dim = q_heads, kv_heads, dim
        self.qkv = torch.randn(width, (q_heads + 2 * kv_heads) * dim, device=device, dtype=torch.bfloat16) * width ** -0.5
        self.out = torch.randn(q_heads * dim, width, device=device, dtype=torch.bfloat16) * (q_heads * dim) ** -0.5
        self.q_weight, self.k_weight = torch.ones(2, dim, device=device).unbind()
        angle = torch.arange(places, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(dim // 2, device=device, dtype=torch.float64) / (dim // 2))
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def write(self, x, cache, pos, crd, row, place):
        """Queries of the tokens x; their keys and values go to the cache."""
        qkv = (x @ self.qkv).view(len(x), -1, self.dim)
        q, k, v = qkv.split([self.q_heads, self.kv_heads, self.kv_heads], 1)
        return cache.append_norm_rope(q, k, v, self.q_weight, self.k_weight, self.cos, self.sin, pos, crd, row, place)

    def step(self, x, cache, pos, crd, row, length):
        """One new token of each request, the last of its `length`."""
        q = self.write(x, cache, pos, crd, row, length - 1)
        return attention.paged_attention(q, cache, pos, crd, length).flatten(1) @ self.out, q


def serve(requests=16, prompt=1000, steps=32, q_heads=32, kv_heads=8, dim=128, width=1024, page_size=64, cache_type=torch.bfloat16, device="cuda"):
    """Runs the loop; returns (microseconds of a step, largest error of the attention, the bound it is held to)."""
    torch.manual_seed(0)
    lens = [max(1, prompt - 37 * r % prompt) for r in range(requests)]  # prompts of different lengths
    layer = Layer(width, q_heads, kv_heads, dim, max(lens) + steps, device)
    each = [-(-(n + steps) // page_size) for n in lens]
    cache = attention.PagedCache.empty(sum(each), kv_heads, page_size, dim, cache_type, device)
    i32 = dict(device=device, dtype=torch.int32)
    pos = torch.tensor([0] + each, **i32).cumsum(0, dtype=torch.int32)
    crd = torch.randperm(sum(each), device=device).int()
    row = torch.arange(requests, **i32)

    tokens = torch.cat([torch.arange(n) for n in lens]).to(**i32)
    layer.write(torch.randn(len(tokens), width, device=device, dtype=torch.bfloat16), cache, pos, crd,
                torch.repeat_interleave(row, torch.tensor(lens, device=device)), tokens)

    x, length = torch.randn(requests, width, device=device, dtype=torch.bfloat16), torch.tensor(lens, **i32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # once outside the capture; the captured step writes the same token again
        layer.step(x, cache, pos, crd, row, length + 1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        length += 1
        y, q = layer.step(x, cache, pos, crd, row, length)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(steps):
        graph.replay()
        x.copy_(y)  # the next token of this example is what the layer said
    end.record()
    torch.cuda.synchronize()

    worst = bound = 0.0
    out = attention.paged_attention(q, cache, pos, crd, length)
    for r, n in enumerate(length.tolist()):
        k, v = cache.read(pos, crd, torch.full((n,), r, **i32), torch.arange(n, **i32), dtype=torch.float32)
        k, v = (t.double().repeat_interleave(q_heads // kv_heads, 1) for t in (k, v))
        p = torch.softmax(torch.einsum("hd,nhd->hn", q[r].double(), k) * dim ** -0.5, -1)
        want = torch.einsum("hn,nhd->hd", p, v)
        worst = max(worst, float((out[r].double() - want).abs().max()))
        bound = max(bound, 2.0 ** -7 * float(want.abs().max()))  # a rounding to bfloat16, and as much for the sums
    return begin.elapsed_time(end) * 1e3 / steps, worst, bound


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=1000)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--cache", choices=("bfloat16", "int8", "float8_e4m3fn"), default="bfloat16")
    args = ap.parse_args()
    us, error, most = serve(args.requests, args.prompt, args.steps, cache_type=getattr(torch, args.cache))
    print(f"{args.requests} requests, prompts of up to {args.prompt} tokens, {args.cache} cache: {us:.1f} us a step, error {error:.2g} (bound {most:.2g})")
    sys.exit(0 if error <= most else 1)
