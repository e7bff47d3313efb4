"""Products with 4-bit weights, and the layer that they are part of (lapis_b200/experts.py), against plain implementations in 64 bits.

Bounds: E = 2^-24 is half a unit in the last place of 32 bits.  Products of a code and a value are exact; sums on the tensor cores
cut what lies below the largest term's last place instead of rounding, 4 E of the terms' magnitudes for each of them; scales and
shares add a rounding each.  ``U`` is the rounding to the result's type.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -120, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -120}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEV = "cuda"


@pytest.fixture(scope="module")
def X():
    from lapis_b200 import experts
    return experts


def normal(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape)).to(DEV)


def weights4(seed, experts, outputs, columns, group, zeros, scale_type):
    rng = np.random.default_rng(seed)
    lead = (outputs,) if experts is None else (experts, outputs)
    groups = -(-columns // group)
    codes = torch.from_numpy(rng.integers(0, 256, (*lead, (columns + 1) // 2), dtype=np.uint8)).to(DEV)
    scale = torch.from_numpy(rng.uniform(-0.1, 0.3, (*lead, groups))).to(DEV, scale_type)
    zero = torch.from_numpy(rng.integers(0, 16, (*lead, groups), dtype=np.uint8)).to(DEV) if zeros else None
    return codes, scale, zero


def dense(codes, scale, zero, columns, group):
    c = torch.arange(columns, device=DEV)
    code = (codes[..., c // 2].int() >> (4 * (c % 2)).int()) & 15
    return (code - (8 if zero is None else zero[..., c // group].int())).double() * scale.double()[..., c // group]


def product(x, w, gated, dtype):
    """The product and how far it may be off in front of its rounding."""
    terms = w.shape[-1] + 32
    y, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    off = 4 * E * terms * size
    if gated:
        a, b = y.chunk(2, -1)
        da, db = off.chunk(2, -1)
        s = a * torch.sigmoid(a)
        y, off = s * b, 1.1 * da * (b.abs() + db) + s.abs() * db + 16 * E * (s * b).abs()  # silu's slope is below 1.1
    return y, off + U[dtype] * y.abs() + TINY[dtype]


PRODUCTS = [
    # rows, outputs, columns, group, zeros, type of scales
    (1, 16, 64, 32, False, "same"), (1, 2, 1, 128, True, F32), (3, 34, 100, 64, False, F32), (8, 130, 257, 32, True, "same"), (9, 48, 256, 128, True, BF16),
    (2, 1000, 1001, 64, True, "same"), (16, 64, 2048, 128, False, F16), (17, 66, 640, 32, False, F32), (33, 160, 2500, 64, True, "same"),
    (64, 128, 1088, 128, True, F32), (65, 32, 320, 32, False, "same"), (130, 18, 192, 64, False, "same"), (5, 20_000, 64, 128, False, "same"),
    (21, 9000, 320, 32, True, F32), (1, 96, 9000, 128, False, "same"), (40, 30, 5001, 64, True, F16),
]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("rows,outputs,columns,group,zeros,scale", PRODUCTS)
def test_product(X, rows, outputs, columns, group, zeros, scale, dtype, gated):
    given = weights4(rows + columns, None, outputs, columns, group, zeros, dtype if scale == "same" else scale)
    matrix = X.Int4Matrix(*given, columns=columns, group=group, gated=gated)
    x = (normal(1, rows, columns) * columns ** -0.5).to(dtype)
    y = matrix.matmul(x)
    want, bound = product(x, dense(*given, columns, group), gated, dtype)
    assert y.dtype == dtype and y.shape == want.shape and y.is_contiguous()
    assert bool(((y.double() - want).abs() <= bound).all())
    assert torch.equal(y, matrix.matmul(x))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
def test_product_of_views(X, dtype):
    given = weights4(3, None, 40, 136, 32, True, dtype)
    matrix = X.Int4Matrix(*given, columns=136, group=32)
    wide = normal(2, 14, 400).to(dtype)
    for x in (wide[:, 8:144], wide[:, 3:139], wide[::2, :136], wide[:1, 5:141].expand(6, 136)):
        assert torch.equal(matrix.matmul(x), matrix.matmul(x.contiguous()))
    assert matrix.matmul(wide[:0, :136]).shape == (0, 40)


def test_32_bits_are_kept(X):
    """Values of 24 bits times codes that pick one column each: what comes out is the value itself, from the largest number to 2^-100."""
    columns = 64
    codes = torch.full((columns, columns // 2), 0x88, dtype=torch.uint8, device=DEV)
    for n in range(columns):
        codes[n, n // 2] = 0x89 if n % 2 == 0 else 0x98  # w = identity
    matrix = X.Int4Matrix(codes, torch.ones(columns, 1, device=DEV), None, columns=columns, group=128)
    x = torch.empty(5, columns, device=DEV).uniform_(-1, 1, generator=torch.Generator(DEV).manual_seed(1))
    x[1] *= 2.0 ** 127
    x[2] *= 2.0 ** -100
    x[3] = torch.finfo(F32).max
    x[4, 0], x[4, 1:] = -torch.finfo(F32).max, 1 + 2.0 ** -23
    assert torch.equal(matrix.matmul(x), x)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
def test_infinities_and_nan_stay_in_their_row(X, dtype):
    given = weights4(5, None, 24, 96, 32, False, F32)
    given[0].fill_(0x99)  # every weight is the scale
    matrix = X.Int4Matrix(*given, columns=96, group=32)
    x = normal(3, 12, 96).to(dtype)
    clean = matrix.matmul(x)
    x[3, 50], x[7, 2] = math.inf, math.nan
    y = matrix.matmul(x)
    keep = [r for r in range(12) if r not in (3, 7)]
    assert torch.equal(y[keep], clean[keep])
    assert torch.equal(y[3].float(), math.inf * given[1][:, 1].sign()) and bool(y[7].isnan().all())


LISTED = [
    # tokens, k, experts, outputs, columns, group, zeros
    (1, 2, 4, 32, 64, 32, False), (7, 3, 5, 50, 100, 64, True), (40, 4, 3, 64, 320, 128, False), (90, 3, 2, 20, 200, 32, True), (3, 8, 60, 130, 72, 128, True),
    (1, 1, 1, 16, 64, 64, False), (64, 8, 128, 48, 256, 32, False),
]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("fetch", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("tokens,k,experts,outputs,columns,group,zeros", LISTED)
def test_product_of_lists(X, tokens, k, experts, outputs, columns, group, zeros, dtype, fetch, gated):
    given = weights4(tokens, experts, outputs, columns, group, zeros, dtype)
    matrix = X.Int4Matrix(*given, columns=columns, group=group, gated=gated)
    expert = torch.from_numpy(np.random.default_rng(tokens + 1).integers(-1, experts + 1, (tokens, k))).to(DEV)
    lists = X.ExpertLists(expert, experts)
    x = (normal(2, tokens if fetch else tokens * k, columns) * columns ** -0.5).to(dtype)
    y = matrix.matmul(x, lists, fetch=fetch)
    w = dense(*given, columns, group)
    rows = x[lists.crd.long() // k] if fetch else x
    pos = lists.pos.tolist()
    assert y.shape == (tokens * k, outputs // 2 if gated else outputs) and not y[pos[-1]:].any()
    for e in range(experts):
        want, bound = product(rows[pos[e]:pos[e + 1]], w[e], gated, dtype)
        assert bool(((y[pos[e]:pos[e + 1]].double() - want).abs() <= bound).all())


def test_bad_lists_are_not_followed(X):
    matrix = X.Int4Matrix(*weights4(1, 4, 32, 64, 32, False, BF16), columns=64, group=32)
    lists = X.ExpertLists(torch.zeros(6, 2, dtype=torch.int32, device=DEV), 4)
    x = normal(2, 6, 64).to(BF16)
    lists.crd = torch.from_numpy(np.random.default_rng(4).integers(-2 ** 31, 2 ** 31 - 1, 12)).to(DEV, torch.int32)
    matrix.matmul(x, lists, fetch=True)
    for pos in ([-7, 2 ** 31 - 1, -2 ** 31, 5, 2 ** 31 - 1], [20, 30, 40, 50, 60], [12, 6, 3, 1, -4]):
        lists.pos = torch.tensor(pos, dtype=torch.int32, device=DEV)
        matrix.matmul(x, lists, fetch=True)
    torch.cuda.synchronize()


def quantised(w, group, zeros, scale_type):
    """Codes, scales and zeros in plain torch, the same operations."""
    columns = w.shape[-1]
    groups = -(-columns // group)
    x = torch.zeros(*w.shape[:-1], groups * group, device=DEV)
    x[..., :columns] = w.float()
    x = x.unflatten(-1, (groups, group))
    if zeros:
        low, high = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
        scale = (0.5 * high - 0.5 * low) / torch.full_like(low, 7.5)
    else:
        scale = x.abs().amax(-1, keepdim=True) / torch.full_like(x[..., :1], 7.0)
    scale = scale.to(scale_type)
    s = scale.float()
    usable = (s > 0) & s.isfinite()
    zero = torch.where(usable, (-low / s).round().clamp(max=15), 0.0) if zeros else torch.full_like(s, 8.0)
    code = torch.where(usable, (x / s).round() + zero, zero).clamp(0 if zeros else 1, 15)
    code = code.flatten(-2)[..., :columns].to(torch.uint8)
    if columns % 2:
        code = torch.cat([code, torch.zeros_like(code[..., :1])], -1)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.squeeze(-1), zero.squeeze(-1).to(torch.uint8) if zeros else None


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype,scale", [(F32, F32), (F32, BF16), (F16, F16), (BF16, BF16), (BF16, F32)], ids=str)
@pytest.mark.parametrize("shape,group", [((1, 1), 32), ((5, 64), 32), ((3, 7, 100), 64), ((40, 1001), 128), ((2, 300, 256), 128)])
def test_quantise(X, shape, group, dtype, scale, zeros):
    w = normal(1, *shape).to(dtype)
    w[..., 0, :40] = 0  # a group of zeros
    if shape[-2] > 2:
        w[..., 1, :] = w[..., 1, :].abs() + 1  # all of one sign
    for got, want in zip(X.quantise_int4(w, group, zeros, scale), quantised(w, group, zeros, scale)):
        assert (got is None) == (want is None) and (got is None or (got.dtype == want.dtype and torch.equal(got, want)))


def test_quantised_weights_are_near(X):
    w = normal(1, 3, 64, 500).to(BF16)
    for zeros, steps in ((False, 7), (True, 7.5)):
        codes, scale, zero = X.quantise_int4(w, 32, zeros, F32)
        got = dense(codes, scale, zero, 500, 32)
        half = scale.double().repeat_interleave(32, -1)[..., :500] * (0.5 + 2.0 ** -20)
        if zeros:
            half = half * 2  # the zero is rounded too
        assert bool(((got - w.double()).abs() <= half).all())
        eye = torch.eye(500, device=DEV, dtype=BF16)
        first = X.Int4Matrix(codes[0].contiguous(), scale[0].contiguous(), None if zero is None else zero[0].contiguous(), columns=500, group=32)
        assert torch.equal(first.matmul(eye).T.float(), got[0].to(BF16).float())


def test_quantise_what_is_not_finite(X):
    w = normal(2, 4, 96).float()
    w[1, 40], w[2, 70] = math.inf, math.nan
    for zeros in (False, True):
        codes, scale, zero = X.quantise_int4(w, 32, zeros)
        assert scale.isnan().nonzero().tolist() == [[1, 1], [2, 2]]
    big = torch.tensor([[3e38, -3e38]], device=DEV)
    assert bool(X.quantise_int4(big, 32, True)[1].isfinite().all())


# ---- as they are used together ------------------------------------------------------


class Layer:
    """Router, gated experts in 4 bits and their way back: a serving step."""

    def __init__(self, X, width, hidden, experts, k, dtype, seed=1):
        self.X, self.experts, self.k, self.hidden = X, experts, k, hidden
        self.gate = (normal(seed, experts, width) * width ** -0.5).to(dtype)
        self.up_given = weights4(seed + 1, experts, 2 * hidden, width, 64, True, dtype)
        self.down_given = weights4(seed + 2, experts, width, hidden, 32, False, dtype)
        self.up = X.Int4Matrix(*self.up_given, columns=width, group=64, gated=True)
        self.down = X.Int4Matrix(*self.down_given, columns=hidden, group=32)

    def __call__(self, x, logits):
        weights, expert = self.X.route(logits, self.k)
        lists = self.X.ExpertLists(expert, self.experts)
        h = self.up.matmul(x, lists, fetch=True)
        return lists.combine(self.down.matmul(h, lists), weights), h, lists, weights


def check_layer(layer, x, logits, out, h, lists, weights):
    """Every stage from what the stage in front of it gave."""
    pos, dtype = lists.pos.tolist(), x.dtype
    chosen = torch.sort(logits.double(), dim=-1, descending=True, stable=True).indices[:, :layer.k]
    assert lists.crd.tolist() == listed_experts(chosen)
    up, down = (dense(*g, n, s) for g, n, s in ((layer.up_given, x.shape[1], 64), (layer.down_given, layer.hidden, 32)))
    total, off = torch.zeros(x.shape, dtype=torch.float64, device=DEV), torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    token = lists.crd.long() // layer.k
    rows, row_off = torch.zeros(len(token), x.shape[1], dtype=torch.float64, device=DEV), torch.zeros(len(token), x.shape[1], dtype=torch.float64, device=DEV)
    for e in range(layer.experts):
        a, b = pos[e], pos[e + 1]
        want, bound = product(x[token[a:b]], up[e], True, dtype)
        assert bool(((h[a:b].double() - want).abs() <= bound).all())
        rows[a:b], row_off[a:b] = product(h[a:b], down[e], False, dtype)
    for j in range(layer.k):
        w = weights[:, j:j + 1].double()
        total += w * rows[lists.place[:, j].long()]
        off += w * row_off[lists.place[:, j].long()] * (1 + layer.k * E)
    bound = off + U[dtype] * total.abs() + layer.k * E * (total.abs() + off) + TINY[dtype] + 2.0 ** -20 * off
    assert bool(((out.double() - total).abs() <= bound + U[dtype] * off).all())


def listed_experts(expert):
    return np.argsort(expert.cpu().numpy().reshape(-1), kind="stable").tolist()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("tokens", [1, 30, 200])
def test_layer(X, tokens, dtype):
    layer = Layer(X, 192, 80, 12, 3, dtype)
    x = (normal(4, tokens, 192) * 0.1).to(dtype)
    logits = x @ layer.gate.T
    check_layer(layer, x, logits, *layer(x, logits))


def test_layer_in_a_graph_and_on_other_streams(X):
    layer = Layer(X, 256, 64, 16, 4, BF16)
    x = (normal(4, 33, 256) * 0.1).to(BF16)
    logits = x.float() @ layer.gate.T.float()
    want = layer(x, logits)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(x, logits)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = layer(x, logits)
        graphs.append((g, res))
    for turn in range(3):  # other tokens in the same tensors, both graphs by turns
        x.copy_(normal(5 + turn, 33, 256) * 0.1)
        logits.copy_(x.float() @ layer.gate.T.float())
        for g, res in graphs:
            g.replay()
            check_layer(layer, x, logits, *res)


def test_lists_of_many_slots_in_a_graph(X):
    """Two launches and a workspace, replayed."""
    expert = torch.from_numpy(np.random.default_rng(1).integers(0, 60, (9000, 4))).to(DEV, torch.int32)
    X.ExpertLists(expert, 60)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lists = X.ExpertLists(expert, 60)
        graphs.append((g, lists))
    for turn in range(2):
        expert.copy_(torch.from_numpy(np.random.default_rng(2 + turn).integers(0, 60, (9000, 4))))
        for g, lists in graphs:
            g.replay()
            assert lists.crd.tolist() == listed_experts(expert)


def test_packing_under_capture_is_refused(X):
    from lapis_b200._lib import LapisError
    given = weights4(1, None, 32, 64, 32, False, BF16)
    x = torch.zeros(1, 64, dtype=BF16, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(LapisError, match="capture"):
            X.Int4Matrix(*given, columns=64, group=32)
        x += 1
    g.replay()
    assert float(x.sum()) == 64.0


def test_training_step(X):
    """Forward and backward of a layer of experts, its products in torch, against autograd in 64 bits."""
    tokens, width, hidden, experts, k = 50, 24, 16, 6, 2
    x, gate, w = normal(1, tokens, width), normal(2, experts, width), normal(3, experts, hidden, width) * width ** -0.5
    g = normal(4, tokens, hidden)
    leaves = [t.clone().requires_grad_() for t in (x, gate, w)]
    logits = leaves[0] @ leaves[1].T
    top = logits.topk(k, -1)
    p = torch.softmax(top.values, -1)
    out64 = torch.einsum("tk,tkh->th", p, torch.einsum("tkhw,tw->tkh", leaves[2][top.indices], leaves[0]))
    want = torch.autograd.grad((out64 * g).sum(), leaves)

    x, gate, w, g = (t.float() for t in (x, gate, w, g))
    logits = x @ gate.T
    weights, expert = X.route(logits, k)
    assert torch.equal(expert.long(), top.indices)
    lists = X.ExpertLists(expert, experts)
    pos = lists.pos.tolist()
    spans = [(e, slice(pos[e], pos[e + 1])) for e in range(experts)]
    rows_in = lists.gather(x)
    rows = torch.cat([rows_in[s] @ w[e].T for e, s in spans])
    out = lists.combine(rows, weights)
    drows, dweights = lists.combine_backward(g, rows, weights)
    dw = torch.stack([drows[s].T @ rows_in[s] for e, s in spans])
    dlogits = X.route_backward(dweights, logits, expert)
    dx = lists.gather_backward(torch.cat([drows[s] @ w[e] for e, s in spans])) + dlogits @ gate
    for got, ref in ((out, out64), (dx, want[0]), (dlogits.T @ x, want[1]), (dw, want[2])):
        # sums of at most a few hundred terms below 10, through three products: 1e-6 of the largest result and a margin of 20
        assert float((got.double() - ref).abs().max()) <= 2e-5 * float(ref.abs().max())
