"""Router, lists, rows there and back (lapis_b200/experts.py) against plain implementations in 64 bits.

Bounds: every result is computed in 32 bits and rounded once.  E = 2^-24 is half a unit in the last place of 32 bits; a
sum of n terms is off by at most n E of the sum of their magnitudes, in any order.  ``U`` is the rounding to the result's type.
expf is off by two units in the last place at most (4 E of the result), and by as much as its argument is off.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEV = "cuda"


@pytest.fixture(scope="module")
def X():
    from lapis_b200 import experts
    return experts


def normal(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape)).to(DEV)


# ---- router -------------------------------------------------------------------


ROUTE = [(1, 1, 1), (1, 64, 6), (3, 5, 5), (37, 130, 5), (64, 256, 8), (17, 1024, 32), (129, 33, 32), (5, 1000, 1), (2, 257, 3), (9, 31, 0)]


def chosen64(logits, k, normalise):
    x = logits.double()
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    values, expert = order.values[:, :k], order.indices[:, :k]
    none = values == -math.inf
    total = torch.logsumexp(values if normalise and k else x, -1, keepdim=True)
    return torch.where(none, 0.0, torch.exp(values - total)), torch.where(none, -1, expert).int()


def weight_error(logits, k, normalise):
    """How far a weight may be off, relative to it: exp's argument and result, of it and of the sum; the sum's additions; the quotient."""
    x = logits.double()
    x = torch.where(x == -math.inf, math.nan, x)
    spread = torch.nan_to_num(x.nan_to_num(-math.inf).amax(-1, keepdim=True) - x, 0.0).amax(-1, keepdim=True)
    return (2 * spread + 8 + logits.shape[1] / 32 + 8 + 2) * E


def masked(seed, tokens, experts, dtype):
    """Some experts switched off, the last token without any."""
    x = 3 * normal(seed, tokens, experts)
    x[torch.from_numpy(np.random.default_rng(seed + 1).random((tokens, experts)) < 0.2).to(DEV)] = -math.inf
    if tokens > 1:
        x[-1] = -math.inf
    return x.to(dtype)


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("tokens,experts,k", ROUTE)
def test_route(X, tokens, experts, k, dtype, normalise):
    for logits in (3 * normal(1, tokens, experts), masked(2, tokens, experts, dtype), normal(3, tokens, experts).round()):  # the last with ties
        logits = logits.to(dtype)
        weights, expert = X.route(logits, k, normalise=normalise)
        want, want_expert = chosen64(logits, k, normalise)
        assert weights.dtype == F32 and expert.dtype == torch.int32 and weights.shape == expert.shape == (tokens, k)
        assert torch.equal(expert, want_expert)
        assert bool(((weights.double() - want).abs() <= want * weight_error(logits, k, normalise) + TINY[F32]).all())


def test_route_takes_any_row_stride(X):
    wide = normal(4, 21, 200).to(BF16)
    for view in (wide[:, 3:63], wide[::2, :64], wide[:1].expand(9, 200)):
        got, want = X.route(view, 4), X.route(view.contiguous(), 4)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        g = normal(5, view.shape[0], 4).float()
        assert torch.equal(X.route_backward(g, view, got[1]), X.route_backward(g, view.contiguous(), got[1]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
def test_route_values_at_the_ends(X, dtype):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    inf, nan = math.inf, math.nan
    logits = torch.tensor([[low, -inf, low, -inf],     # the lowest number of a type is chosen like any other
                           [high, low, -inf, 0.0],
                           [0.0, -0.0, 0.0, -0.0],     # equal
                           [1.0, inf, 0.0, -1.0],
                           [1.0, 2.0, nan, 3.0],
                           [-inf, -inf, -inf, 5.0]], dtype=dtype, device=DEV)
    weights, expert = X.route(logits, 2)
    assert expert.tolist() == [[0, 2], [0, 3], [0, 1], [1, 0], [2, 3], [3, -1]]
    assert weights[0].tolist() == weights[2].tolist() == [0.5, 0.5] and weights[1].tolist() == [1.0, 0.0]
    assert bool(weights[4].isnan().all()) and bool(weights[3].isnan().any()) and weights[5].tolist() == [1.0, 0.0]
    all_of, same = X.route(logits, 2, normalise=False)
    assert torch.equal(same, expert) and all_of[0].tolist() == [0.5, 0.5] and all_of[2].tolist() == [0.25, 0.25]
    g = torch.ones(6, 2, device=DEV)
    for normalise in (True, False):
        d = X.route_backward(g, logits, expert, normalise=normalise)
        assert bool(d[[0, 1, 2, 5]].isfinite().all()) and bool(d[4].isnan().any())


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("tokens,experts,k", ROUTE)
def test_route_backward(X, tokens, experts, k, dtype, normalise):
    for logits in ((3 * normal(1, tokens, experts)).to(dtype), masked(2, tokens, experts, dtype)):
        expert = X.route(logits, k)[1]
        g = normal(6, tokens, k).float()
        got = X.route_backward(g, logits, expert, normalise=normalise)
        assert got.dtype == dtype and got.shape == logits.shape and got.is_contiguous()
        here, at = expert >= 0, expert.clamp(min=0).long()
        x = logits.double()
        most = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(most == -math.inf, 0.0, most))
        mine = torch.where(here, e.gather(-1, at), 0.0)
        total = (mine if normalise else e).sum(-1, keepdim=True)
        total = torch.where(total == 0, 1.0, total)
        w, p = mine / total, torch.zeros_like(e) if normalise else e / total
        inner, size = (w * g).sum(-1, keepdim=True), (w * g.abs()).sum(-1, keepdim=True)
        own = torch.where(here, w * (g - inner) if normalise else w * g, 0.0)
        want = torch.zeros_like(x).scatter_add(-1, at, own) - p * inner
        scale = torch.zeros_like(x).scatter_add(-1, at, torch.where(here, w * (g.abs() + size), 0.0)) + p * size
        # the weights' errors count twice, in w and in the inner product, which adds k numbers of its own
        bound = U[dtype] * want.abs() + TINY[dtype] + (2 * weight_error(logits, k, normalise) + (k + 8) * E) * scale
        assert bool(((got.double() - want).abs() <= bound).all())
        assert torch.equal(got, X.route_backward(g, logits, expert, normalise=normalise))


@pytest.mark.parametrize("normalise", [True, False])
def test_route_backward_against_differences(X, normalise):
    logits = normal(7, 6, 12).float()
    weights, expert = X.route(logits, 3, normalise=normalise)
    g, step = normal(8, 6, 3).float(), 1e-4

    def f(x):  # the weights of the same choice, in 64 bits
        e = x.double().exp()
        mine = e.gather(-1, expert.long())
        return (mine / (mine if normalise else e).sum(-1, keepdim=True) * g).sum()
    got = X.route_backward(g, logits, expert, normalise=normalise)
    for i in range(6):
        for j in range(12):
            d = torch.zeros(6, 12, device=DEV, dtype=torch.float64)
            d[i, j] = step
            slope = float(f(logits.double() + d) - f(logits.double() - d)) / (2 * step)
            assert abs(slope - float(got[i, j])) <= 1e-6  # third derivatives are below 6, times step^2; 32 bits leave 1e-7 x 4


def test_route_backward_of_experts_named_twice_or_outside(X):
    logits = normal(9, 1, 5).float().expand(3, 5).contiguous()
    expert = torch.tensor([[2, 2], [2, 7], [-1, -9]], dtype=torch.int32, device=DEV)
    g = torch.tensor([[1.0, 3.0], [4.0, 5.0], [1.0, 2.0]], device=DEV)
    d = X.route_backward(g, logits, expert, normalise=False)
    p = torch.softmax(logits[0].double(), -1)
    want = torch.stack([4.0 * p[2] * (torch.eye(5, device=DEV)[2] - p)] * 2 + [0 * p])
    assert bool(((d.double() - want).abs() <= 60 * E * 8).all())
    assert not X.route_backward(g, logits, expert)[1:].any()  # one choice has the weight 1, whatever its logit


# ---- lists ----------------------------------------------------------------------


def listed(expert, experts):
    e = expert.cpu().numpy().reshape(-1).astype(np.int64)
    e = np.where((e < 0) | (e >= experts), experts, e)
    crd = np.argsort(e, kind="stable")
    place = np.empty_like(crd)
    place[crd] = np.arange(len(crd))
    pos = np.concatenate([[0], np.cumsum(np.bincount(e, minlength=experts + 1))])[:experts + 1]
    return pos, crd, place.reshape(expert.shape)


def same_lists(lists, expert, experts):
    for got, want in zip((lists.pos, lists.crd, lists.place), listed(expert, experts)):
        assert got.dtype == torch.int32 and got.is_contiguous() and np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("tokens,k,experts", [(0, 3, 4), (5, 0, 4), (1, 1, 1), (1, 1, 0), (7, 5, 3), (64, 8, 64), (171, 3, 128), (513, 1, 1024), (2500, 2, 7),
                                              (9000, 8, 60), (10_001, 8, 256), (20_003, 8, 1024), (40_000, 8, 128), (88_000, 8, 33)])
def test_lists(X, tokens, k, experts, index):
    rng = np.random.default_rng(tokens + k)
    expert = torch.from_numpy(rng.integers(-1, experts + 1, (tokens, k))).to(DEV, index)
    same_lists(X.ExpertLists(expert, experts), expert, experts)


@pytest.mark.parametrize("slots", [1000, 30_000, 200_000])
def test_lists_of_one_expert_and_of_none(X, slots):
    for value, experts in ((3, 9), (-5, 9), (2 ** 40 + 1, 9), (0, 1)):
        expert = torch.full((slots, 1), value, dtype=torch.int64, device=DEV)
        same_lists(X.ExpertLists(expert, experts), expert, experts)


# ---- rows there and back ----------------------------------------------------------


ROWS = [(1, 1, 1, 1), (3, 2, 4, 7), (5, 8, 6, 8), (33, 3, 5, 100), (40, 4, 60, 2056), (17, 11, 3, 1001), (9, 33, 50, 64), (6, 40, 9, 130), (301, 8, 16, 512),
        (4, 2, 3, 5000)]


def strided(x, how):
    """The same rows, laid out otherwise."""
    if how == "no":
        return x.contiguous()
    if how == "padded":  # rows at multiples of 16 bytes
        w = torch.zeros(x.shape[0], (x.shape[1] + 23) // 8 * 8, dtype=x.dtype, device=DEV)
        w[:, 8:8 + x.shape[1]] = x
        return w[:, 8:8 + x.shape[1]]
    w = torch.zeros(x.shape[0], x.shape[1] + 3, dtype=x.dtype, device=DEV)
    w[:, 1:1 + x.shape[1]] = x
    return w[:, 1:1 + x.shape[1]]


def some_lists(X, tokens, k, experts):
    expert = torch.from_numpy(np.random.default_rng(tokens * k).integers(-1, experts + 1, (tokens, k))).to(DEV)
    lists = X.ExpertLists(expert, experts)
    here = (lists.place < lists.pos[-1])
    return lists, here


@pytest.mark.parametrize("how", ["no", "padded", "odd"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("tokens,k,experts,dim", ROWS)
def test_gather(X, tokens, k, experts, dim, dtype, how):
    lists, here = some_lists(X, tokens, k, experts)
    x = strided(normal(1, tokens, dim).to(dtype), how)
    rows = lists.gather(x)
    want = torch.zeros(tokens * k, dim, dtype=dtype, device=DEV)
    want[lists.place.long()] = torch.where(here[..., None], x[:, None], 0.0)
    assert rows.is_contiguous() and torch.equal(rows, want)


@pytest.mark.parametrize("how", ["no", "padded", "odd"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("tokens,k,experts,dim", ROWS)
def test_combine_and_backward(X, tokens, k, experts, dim, dtype, how):
    lists, here = some_lists(X, tokens, k, experts)
    rows = normal(2, tokens * k, dim).to(dtype)
    rows[int(lists.pos[-1]):] = math.nan  # of no expert: not looked at
    rows, dout = strided(rows, how), strided(normal(3, tokens, dim).to(dtype), how)
    weights = normal(4, tokens, k).float()
    mine = torch.where(here[..., None], rows[lists.place.long()].double(), 0.0)
    for got, w in ((lists.combine(rows, weights), weights.double()), (lists.gather_backward(rows), torch.ones_like(weights).double())):
        want, size = torch.einsum("tkd,tk->td", mine, w), torch.einsum("tkd,tk->td", mine.abs(), w.abs())
        assert got.dtype == dtype and got.shape == (tokens, dim) and got.is_contiguous()
        assert bool(((got.double() - want).abs() <= U[dtype] * want.abs() + TINY[dtype] + (k + 1) * E * size).all())
    drows, dweights = lists.combine_backward(dout, rows, weights)
    want = torch.zeros(tokens * k, dim, dtype=torch.float64, device=DEV)
    want[lists.place.long()] = torch.where(here[..., None], dout[:, None].double() * weights[..., None].double(), 0.0)
    assert drows.dtype == dtype and bool(((drows.double() - want).abs() <= (U[dtype] + 2 * E) * want.abs() + TINY[dtype]).all())
    want, size = (mine * dout[:, None].double()).sum(-1), (mine * dout[:, None].double()).abs().sum(-1)
    assert dweights.dtype == F32 and bool(((dweights.double() - want).abs() <= (dim + 1) * E * size + TINY[F32]).all())
    assert torch.equal(lists.combine(rows, weights), lists.combine(rows, weights))


def test_gradients_against_differences(X):
    """Sums of products: a difference of two results over a step of any size is the slope."""
    lists, _ = some_lists(X, 19, 3, 5)
    rows, weights, x = normal(5, 57, 40).float(), normal(6, 19, 3).float(), normal(7, 19, 40).float()
    g, d = normal(8, 19, 40).float(), normal(9, 57, 40).float()
    drows, dweights = lists.combine_backward(g, rows, weights)

    def inner(a, b):
        return float((a.double() * b.double()).sum())
    slope = inner(lists.combine(rows + d, weights), g) - inner(lists.combine(rows - d, weights), g)
    assert abs(slope / 2 - inner(drows, d)) <= 1e-4
    step = normal(10, 19, 3).float()
    slope = inner(lists.combine(rows, weights + step), g) - inner(lists.combine(rows, weights - step), g)
    assert abs(slope / 2 - inner(dweights, step)) <= 1e-4
    dx = lists.gather_backward(d)
    assert abs((inner(lists.gather(x + g), d) - inner(lists.gather(x - g), d)) / 2 - inner(dx, g)) <= 1e-4  # 760 to 2280 terms of about 1, 1e-7 of each


def test_bad_lists_are_not_followed(X):
    """Places, offsets and slots that point anywhere: nothing is read or written there."""
    lists, _ = some_lists(X, 12, 2, 4)
    x, rows, weights = normal(1, 12, 24).to(BF16), normal(2, 24, 24).to(BF16), normal(3, 12, 2).float()
    lists.place = torch.from_numpy(np.random.default_rng(4).integers(-2 ** 31, 2 ** 31 - 1, (12, 2))).to(DEV, torch.int32)
    lists.gather(x)
    assert not lists.combine(rows, weights).any()
    assert not lists.combine_backward(x, rows, weights)[1].any()
    lists.pos = torch.tensor([-7, 2 ** 31 - 1, -2 ** 31, 5, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    lists.gather(x)
    torch.cuda.synchronize()


def test_rows_behind_32_bits(X):
    """70,000 rows of 40,000 values: offsets beyond 2^31 elements."""
    tokens, dim = 70_000, 40_000
    expert = torch.zeros(tokens, 1, dtype=torch.int32, device=DEV)
    lists = X.ExpertLists(expert, 1)
    x = torch.zeros(tokens, dim, dtype=F16, device=DEV)
    x[:, ::1000] = torch.arange(tokens, device=DEV)[:, None].remainder(2048).to(F16)
    rows = lists.gather(x)
    assert torch.equal(rows, x)
    del x
    out = lists.combine(rows, torch.full((tokens, 1), 2.0, device=DEV))
    assert torch.equal(out[-5:], 2 * rows[-5:]) and torch.equal(out[53_680:53_700], 2 * rows[53_680:53_700])
