"""A layer of experts as the first call of a process, under stream capture: what the calls set up on first use has to be allowed there."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

LAYER = """
import torch
from lapis_b200 import experts as E
torch.manual_seed(0)
tokens, experts, k, width, hidden = {shape}
up = E.Int4Matrix.quantise(torch.randn(experts, 2 * hidden, width, device="cuda", dtype=torch.bfloat16) * width ** -0.5, 64, gated=True)
down = E.Int4Matrix.quantise(torch.randn(experts, width, hidden, device="cuda", dtype=torch.bfloat16) * hidden ** -0.5, 128)
x, logits = torch.randn(tokens, width, device="cuda", dtype=torch.bfloat16), torch.randn(tokens, experts, device="cuda")
def layer():
    weights, expert = E.route(logits, k)
    lists = E.ExpertLists(expert, experts)
    rows = down.matmul(up.matmul(x, lists, fetch=True), lists)
    out = lists.combine(rows, weights)
    drows, dweights = lists.combine_backward(out, rows, weights)
    return out, drows, dweights, E.route_backward(dweights, logits, expert), lists.gather_backward(lists.gather(x))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = layer()
for _ in range(2):
    for t in got:
        t.zero_()
    graph.replay()
    assert all(torch.equal(a, b) and bool(a.any()) for a, b in zip(got, layer()))
print("done")
"""


@pytest.mark.parametrize("shape", [(3, 8, 2, 256, 96), (200, 4, 2, 512, 128), (3000, 16, 2, 128, 64)])
def test_layer_of_experts(shape):
    """Few and many rows of each expert, lists of one block and of several."""
    r = subprocess.run([sys.executable, "-c", LAYER.format(shape=shape)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "done\n", r.stdout + r.stderr[-2000:]
