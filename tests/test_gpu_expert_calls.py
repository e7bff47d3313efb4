"""Calls of a layer of experts at their edges: nothing to do, captured and replayed, two at once, magnitudes of every exponent."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEV = "cuda"


@pytest.fixture(scope="module")
def X():
    from lapis_b200 import experts
    return experts


def normal(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape)).to(DEV)


def random_matrix(X, seed, experts, outputs, columns, group, zeros=False, gated=False, dtype=BF16):
    rng = np.random.default_rng(seed)
    lead = (outputs,) if experts is None else (experts, outputs)
    codes = torch.from_numpy(rng.integers(0, 256, (*lead, (columns + 1) // 2), dtype=np.uint8)).to(DEV)
    groups = -(-columns // group)
    scale = torch.from_numpy(rng.uniform(0.01, 0.1, (*lead, groups))).to(DEV, dtype)
    zero = torch.from_numpy(rng.integers(0, 16, (*lead, groups), dtype=np.uint8)).to(DEV) if zeros else None
    return X.Int4Matrix(codes, scale, zero, columns=columns, group=group, gated=gated)


def test_nothing_to_do(X):
    none = X.ExpertLists(torch.zeros(5, 0, dtype=torch.int32, device=DEV), 4)
    assert none.pos.tolist() == [0] * 5 and none.crd.numel() == 0
    x = normal(1, 5, 48).to(BF16)
    assert none.gather(x).shape == (0, 48)
    out = none.combine(torch.empty(0, 48, dtype=BF16, device=DEV), torch.empty(5, 0, device=DEV))
    assert out.shape == (5, 48) and not out.any()
    lists = X.ExpertLists(torch.zeros(3, 2, dtype=torch.int32, device=DEV), 4)
    narrow = torch.empty(6, 0, dtype=BF16, device=DEV)
    assert lists.gather(narrow[:3]).shape == (6, 0) and lists.combine(narrow, torch.ones(3, 2, device=DEV)).shape == (3, 0)
    drows, dweights = lists.combine_backward(narrow[:3], narrow, torch.ones(3, 2, device=DEV))
    assert drows.shape == (6, 0) and dweights.tolist() == [[0.0, 0.0]] * 3
    weights, expert = X.route(torch.empty(4, 0, device=DEV), 0)
    assert weights.shape == expert.shape == (4, 0)
    empty = X.Int4Matrix(torch.empty(6, 0, dtype=torch.uint8, device=DEV), torch.empty(6, 0, device=DEV), columns=0)
    y = empty.matmul(torch.empty(3, 0, device=DEV))
    assert y.shape == (3, 6) and not y.any()
    matrix = random_matrix(X, 1, 4, 32, 64, 32)
    assert matrix.matmul(torch.empty(0, 64, dtype=BF16, device=DEV), none).shape == (0, 32)


def identity(X, n, dtype):
    """w = 1 on the diagonal: code 9 with a zero of 8 and a scale of 1."""
    codes = torch.full((n, n // 2), 0x88, dtype=torch.uint8, device=DEV)
    i = torch.arange(n, device=DEV)
    codes[i, i // 2] = torch.where(i % 2 == 0, 0x89, 0x98).to(torch.uint8)
    return X.Int4Matrix(codes, torch.ones(n, -(-n // 64), device=DEV), None, columns=n, group=64)


@pytest.mark.parametrize("rows", [1, 8, 9, 40, 70])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
def test_values_of_every_exponent_come_out_as_they_are(X, dtype, rows):
    info = torch.finfo(dtype)
    low, high = math.log2(info.tiny), math.log2(info.max)
    # three parts of a 32-bit value are whole where the last one is a normal bf16
    low += 24 if dtype == F32 else 0
    x = torch.from_numpy(np.exp2(np.random.default_rng(rows).uniform(low, high, (rows, 128))) * np.random.default_rng(1).choice([-1, 1], (rows, 128))).to(DEV, dtype)
    x[0, :2] = torch.tensor([info.max, info.min], dtype=dtype, device=DEV)
    assert bool(x.isfinite().all())
    assert torch.equal(identity(X, 128, dtype).matmul(x), x)


SPLIT = [
    # rows, outputs, columns, group, zeros: few tiles, whose columns a cluster's CTAs share unevenly
    (40, 96, 9000, 128, False), (12, 300, 300, 32, True), (100, 130, 1400, 64, False), (20, 128, 4096, 64, True), (1000, 64, 520, 128, True), (64, 16, 64, 32, False),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("rows,outputs,columns,group,zeros", SPLIT)
def test_shared_tiles(X, rows, outputs, columns, group, zeros, dtype):
    """Rows of a product do not depend on one another: many rows give what each few of them give, but for the order of sums in 32 bits."""
    matrix = random_matrix(X, rows, None, outputs, columns, group, zeros, dtype=F32)
    x = (normal(2, rows, columns) * columns ** -0.5).to(dtype)
    y = matrix.matmul(x)
    some = torch.arange(0, rows, max(1, rows // 24), device=DEV)[:24]
    each = torch.cat([matrix.matmul(x[r:r + 1]) for r in some.tolist()])
    # |w| up to 1.5: both are off by 4 x 2^-24 of the terms' magnitudes for each of them, and rounded once
    size = 1.5 * x[some].double().abs().sum(-1, keepdim=True)
    bound = 2 * 4 * 2.0 ** -24 * (columns + 32) * size + 2 * {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype] * each.double().abs() + 1e-6
    assert bool(((y[some].double() - each.double()).abs() <= bound).all())
    assert torch.equal(y, matrix.matmul(x))


def test_two_streams_at_once(X):
    """Launches whose clusters share tiles, of both amounts of tensor memory, in flight together."""
    matrices = [random_matrix(X, s, None, 512, 4096, g) for s, g in ((1, 128), (2, 32), (3, 64), (4, 128))]
    xs = [(normal(s, r, 4096) / 64).to(BF16) for s, r in ((1, 40), (2, 60), (3, 64), (4, 100))]
    want = [m.matmul(x) for m, x in zip(matrices, xs)]
    streams = [torch.cuda.Stream() for _ in matrices]
    torch.cuda.synchronize()
    got = [[] for _ in matrices]
    for _ in range(25):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(matrices[i].matmul(xs[i]))
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(w, y) for y in ys)


@pytest.mark.parametrize("tokens", [5, 150])
def test_layers_in_two_graphs(X, tokens):
    """Few and many rows of each expert, captured twice and replayed by turns on other values."""
    experts, k, width, hidden = 6, 3, 1024, 320
    up, down = random_matrix(X, 1, experts, 2 * hidden, width, 128, gated=True), random_matrix(X, 2, experts, width, hidden, 32, zeros=True)
    x, logits = (normal(3, tokens, width) / 32).to(BF16), normal(4, tokens, experts).float()

    def layer():
        weights, expert = X.route(logits, k)
        lists = X.ExpertLists(expert, experts)
        return lists.combine(down.matmul(up.matmul(x, lists, fetch=True), lists), weights)
    layer()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer()
        graphs.append((g, out))
    for turn in range(3):
        x.copy_(normal(5 + turn, tokens, width) / 32)
        logits.copy_(normal(9 + turn, tokens, experts))
        want = layer()
        for g, out in graphs:
            out.zero_()
            g.replay()
            assert torch.equal(out, want)


def test_scratch_that_a_graph_cannot_keep_is_refused(X):
    """70,000 rows of 2048 columns are 287 MB as they are laid out, more than the library's pool holds."""
    from lapis_b200._lib import LapisError
    matrix = random_matrix(X, 1, None, 16, 2048, 128)
    x = torch.ones(70_000, 2048, dtype=BF16, device=DEV)
    want = matrix.matmul(x)
    assert torch.equal(want, matrix.matmul(x[:1]).expand(70_000, 16))
    few = matrix.matmul(x[:100])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(LapisError, match="under stream capture"):
            matrix.matmul(x)
        y = matrix.matmul(x[:100])
    y.zero_()
    g.replay()
    assert torch.equal(y, few)


def test_operands_of_the_wrong_kind_on_the_device(X):
    lists = X.ExpertLists(torch.zeros(3, 2, dtype=torch.int32, device=DEV), 4)
    x = torch.zeros(3, 16, dtype=BF16, device=DEV)
    for bad in (x.double(), x[:2], x.reshape(-1), x.t().contiguous().t(), x.cpu()):
        with pytest.raises((TypeError, ValueError), match="x must|x:"):
            lists.gather(bad)
    rows, weights = torch.zeros(6, 16, dtype=BF16, device=DEV), torch.ones(3, 2, device=DEV)
    with pytest.raises(TypeError, match="weights"):
        lists.combine(rows, weights.double())
    with pytest.raises(ValueError, match="weights"):
        lists.combine(rows, weights[:2])
    with pytest.raises(TypeError, match="dout"):
        lists.combine_backward(x.float(), rows, weights)
    lists.crd = lists.crd.long()
    with pytest.raises(TypeError, match="crd"):
        lists.gather(x)
    with pytest.raises(ValueError, match="expert must"):
        X.ExpertLists(torch.zeros(3, dtype=torch.int32, device=DEV), 4)
    with pytest.raises(ValueError, match="between 0 and 1024"):
        X.ExpertLists(torch.zeros(3, 1, dtype=torch.int32, device=DEV), -1)
    with pytest.raises(ValueError, match="k must"):
        X.route(torch.zeros(3, 4, device=DEV), 5)
    matrix = random_matrix(X, 1, 4, 32, 64, 32)
    with pytest.raises(Exception, match="need lists"):
        matrix.matmul(torch.zeros(2, 64, dtype=BF16, device=DEV))
    with pytest.raises(ValueError, match="x must"):
        matrix.matmul(torch.zeros(2, 65, dtype=BF16, device=DEV))
    with pytest.raises(ValueError, match="fetched"):
        matrix.matmul(torch.zeros(2, 64, dtype=BF16, device=DEV), fetch=True)
    for kw in ({"columns": 62}, {"columns": 64, "group": 48}, {"columns": 64, "group": 32}, {"columns": 64, "gated": True}):
        with pytest.raises(ValueError):
            X.Int4Matrix(torch.zeros(7, 32, dtype=torch.uint8, device=DEV), torch.zeros(7, 1, device=DEV), **kw)
