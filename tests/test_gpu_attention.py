"""Norms with rotation, the paged cache and attention of one new token (lapis_b200/attention.py) against plain
implementations in 64 bits.

Bounds: every result is computed in 32 bits and rounded once.  E = 2^-24 is half a unit in the last place of 32 bits; a
sum of n terms is off by at most n E of the sum of their magnitudes, in any order.  ``U`` is the rounding to the result's
type.  Sums of products on the tensor cores cut what lies below the largest term's last place instead of rounding: 4 E.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
#: How far the weights of a softmax may be rounded in front of the product with the values.
WEIGHT = {torch.float32: 0.0, torch.float16: 2.0 ** -16, torch.bfloat16: 2.0 ** -11}
F32, F16, BF16, I8, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn
DEV = "cuda"


@pytest.fixture(scope="module")
def A():
    from lapis_b200 import attention
    return attention


def normal(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape)).to(DEV)


# ---- rotate -----------------------------------------------------------------


def tables(places, rot):
    angle = torch.arange(places, device=DEV)[:, None] * 100.0 ** (-torch.arange(rot // 2, device=DEV) / max(1, rot // 2))
    return angle.double().cos().float().contiguous(), angle.double().sin().float().contiguous()


def pairs(rot, near):
    i = torch.arange(rot // 2, device=DEV)
    return (2 * i, 2 * i + 1) if near else (i, i + rot // 2)


def turn(y, cos, sin, place, near, back=False):
    """Rotated rows; with `back` the other way."""
    a, b = pairs(2 * cos.shape[1], near)
    c, s = cos.double()[place][:, None], sin.double()[place][:, None] * (-1 if back else 1)
    out = y.clone()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    return out


def forward64(x, w, cos, sin, place, eps, near):
    x, w = x.double(), w.double()
    return turn(x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w, cos, sin, place, near)


def partners(y, rot, near):
    """Sum of the magnitudes of the two elements that a rotated one comes from."""
    a, b = pairs(rot, near)
    out = y.abs().clone()
    out[..., a] = out[..., b] = y[..., a].abs() + y[..., b].abs()
    return out


ROTATE = [
    # tokens, q heads, k heads, dim, rot, pairs, type, weights, indices
    (1, 1, 1, 2, 2, "near", F32, F32, torch.int32),
    (3, 2, 1, 128, 128, "half", BF16, BF16, torch.int32),
    (5, 32, 8, 128, 128, "half", BF16, F32, torch.int64),
    (7, 4, 2, 128, 64, "near", F16, F16, torch.int32),
    (2, 3, 1, 128, 32, "half", F32, F32, torch.int32),
    (33, 5, 5, 80, 80, "half", F16, F32, torch.int32),
    (9, 3, 3, 96, 48, "near", F32, F32, torch.int64),
    (4, 6, 2, 256, 256, "half", BF16, BF16, torch.int32),
    (4, 6, 2, 256, 128, "near", F32, F32, torch.int32),
    (17, 8, 1, 64, 64, "near", BF16, F32, torch.int32),
    (6, 2, 2, 72, 72, "half", BF16, BF16, torch.int32),   # half of the pairs end inside 16 bytes
    (6, 2, 2, 7, 4, "half", F32, F32, torch.int32),
    (6, 2, 2, 7, 4, "near", BF16, F32, torch.int32),
    (6, 1, 3, 37, 0, "half", F16, F32, torch.int32),      # norms alone
    (11, 0, 4, 112, 112, "half", BF16, BF16, torch.int32),  # keys alone
    (300, 4, 1, 192, 96, "half", F16, F16, torch.int32),
    (2000, 2, 1, 32, 32, "half", BF16, BF16, torch.int32),
]


def rotate_inputs(c, strided):
    tokens, hq, hk, dim, rot, near, dtype, wtype, idx = c
    x = normal(1, tokens, hq + hk + 3, dim + (3 if strided == "odd" else 0)).to(dtype)
    if strided == "heads first":  # [heads, tokens, dim] seen as [tokens, heads, dim]
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    q, k = x[:, :hq, :dim], x[:, hq:hq + hk, :dim]
    if strided == "no":
        q, k = q.contiguous(), k.contiguous()
    w = (1 + 0.3 * normal(2, 2, dim)).to(wtype)
    cos, sin = tables(50, rot)
    place = torch.from_numpy(np.random.default_rng(3).integers(0, 50, tokens)).to(DEV, idx)
    return q, k, w[0].contiguous(), w[1].contiguous(), cos, sin, place, near == "near"


@pytest.mark.parametrize("strided", ["no", "view", "odd", "heads first"])
@pytest.mark.parametrize("c", ROTATE, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_rotate(A, c, strided):
    q, k, qw, kw, cos, sin, place, near = rotate_inputs(c, strided)
    got = A.qk_norm_rope(q, k, qw, kw, cos, sin, place, eps=1e-5, interleaved=near)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        want = forward64(x, w, cos, sin, place.long(), 1e-5, near)
        n = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        bound = U[x.dtype] * want.abs() + TINY[x.dtype] + (x.shape[2] + 16) * E * partners(n, c[4], near)
        assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
        assert bool(((y.double() - want).abs() <= bound).all())


def backward64(dy, x, w, cos, sin, place, eps, near):
    dy, x, w = dy.double(), x.double(), w.double()
    dn = turn(dy, cos, sin, place, near, back=True)
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    g = dn * w
    return r * (g - x * r * r * (g * x).mean(-1, keepdim=True)), (dn * x * r).sum((0, 1)), dn, r


@pytest.mark.parametrize("strided", ["no", "view", "odd"])
@pytest.mark.parametrize("c", ROTATE, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_rotate_backward(A, c, strided):
    q, k, qw, kw, cos, sin, place, near = rotate_inputs(c, strided)
    dq, dk = normal(5, *q.shape).to(q.dtype), normal(6, *k.shape).to(q.dtype)
    if strided == "odd":
        dq = torch.cat([dq, dq[..., :1]], -1)[..., :-1]
    got = A.qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, place, eps=1e-5, interleaved=near)
    again = A.qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, place, eps=1e-5, interleaved=near)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    for x, w, dy, dx, dw in ((q, qw, dq, got[0], got[2]), (k, kw, dk, got[1], got[3])):
        want, want_w, dn, r = backward64(dy, x, w, cos, sin, place.long(), 1e-5, near)
        dim = x.shape[2]
        g = partners(dy.double(), c[4], near) * w.double().abs()
        size = r * (g + x.double().abs() * r * r * (g * x.double().abs()).mean(-1, keepdim=True))
        bound = U[x.dtype] * want.abs() + TINY[x.dtype] + (2 * dim + 32) * E * size
        assert dx.dtype == x.dtype and bool(((dx.double() - want).abs() <= bound).all())
        terms = (partners(dy.double(), c[4], near) * x.double().abs() * r).sum((0, 1))
        assert dw.dtype == F32 and bool(((dw.double() - want_w).abs() <= (x.shape[0] * x.shape[1] + dim + 32) * E * terms).all())


def test_rotate_backward_against_differences(A):
    """Central differences of the formula in 64 bits: third derivatives are of order one, h = 1e-5 gives about 1e-10."""
    c = (3, 2, 1, 20, 12, "half", F32, F32, torch.int32)
    q, k, qw, kw, cos, sin, place, near = rotate_inputs(c, "no")
    dq, dk = normal(5, *q.shape).float(), normal(6, *k.shape).float()
    got = A.qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, place, eps=1e-5)

    def loss(x, w, dy):
        return float((forward64(x, w, cos, sin, place.long(), 1e-5, near) * dy.double()).sum())

    for x, w, dy, dx, dw in ((q, qw, dq, got[0], got[2]), (k, kw, dk, got[1], got[3])):
        for of, grad in ((x, dx), (w, dw)):
            flat = grad.double().flatten()
            for i in range(0, flat.numel(), 7):
                up, down = of.double().clone(), of.double().clone()
                up.view(-1)[i] += 1e-5
                down.view(-1)[i] -= 1e-5
                d = (loss(up, w, dy) - loss(down, w, dy) if of is x else loss(x, up, dy) - loss(x, down, dy)) / 2e-5
                assert abs(float(flat[i]) - d) <= 1e-5 * (1 + abs(d))


def test_rotate_padding_and_empty(A):
    q, k, qw, kw, cos, sin, place, near = rotate_inputs((6, 2, 1, 64, 64, "half", BF16, BF16, torch.int32), "view")
    place[1], place[4] = -1, 50
    for x in A.qk_norm_rope(q, k, qw, kw, cos, sin, place):
        assert float(x[[1, 4]].abs().max()) == 0 and float(x[[0, 2, 3, 5]].abs().amax(-1).min()) > 0
    whole = A.qk_norm_rope_backward(q, k, q, k, qw, kw, cos, sin, place)
    assert float(whole[0][[1, 4]].abs().max()) == 0 and float(whole[1][[1, 4]].abs().max()) == 0
    keep = [0, 2, 3, 5]
    part = A.qk_norm_rope_backward(q[keep], k[keep], q[keep], k[keep], qw, kw, cos, sin, place[keep])
    assert torch.allclose(whole[2], part[2], rtol=1e-5, atol=1e-5) and torch.allclose(whole[3], part[3], rtol=1e-5, atol=1e-5)
    none = A.qk_norm_rope_backward(q[:0], k[:0], q[:0], k[:0], qw, kw, cos, sin, place[:0])
    assert none[0].shape == (0, 2, 64) and float(none[2].abs().max()) == 0 and float(none[3].abs().max()) == 0
    assert A.qk_norm_rope(q[:0], k[:0], qw, kw, cos, sin, place[:0])[0].shape == (0, 2, 64)


def test_rotate_zero_rows(A):
    """A head of zeros stays one, and its gradient is that of x / sqrt(eps)."""
    q, k, qw, kw, cos, sin, place, near = rotate_inputs((2, 1, 1, 64, 64, "half", F32, F32, torch.int32), "no")
    q.zero_()
    assert float(A.qk_norm_rope(q, k, qw, kw, cos, sin, place, eps=1e-6)[0].abs().max()) == 0
    dq = normal(4, *q.shape).float()
    got = A.qk_norm_rope_backward(dq, k, q, k, qw, kw, cos, sin, place, eps=1e-6)[0]
    want = backward64(dq, q, qw, cos, sin, place.long(), 1e-6, near)[0]
    assert bool(((got.double() - want).abs() <= 1e-5 * want.abs().max()).all())


# ---- the cache --------------------------------------------------------------


def lists(each, pages, seed, idx=torch.int32):
    """CSR page lists: `each[r]` pages for request r, no page twice."""
    perm = np.random.default_rng(seed).permutation(pages)[:sum(each)]
    pos = np.concatenate([[0], np.cumsum(each)])
    return torch.from_numpy(pos).to(DEV, idx), torch.from_numpy(perm).to(DEV, idx)


def tokens_of(lens, idx=torch.int32):
    row = np.repeat(np.arange(len(lens)), lens)
    place = np.concatenate([np.arange(n) for n in lens]) if len(lens) else np.zeros(0)
    return torch.from_numpy(row).to(DEV, idx), torch.from_numpy(place).to(DEV, idx)


def quantised(x, store):
    """What a cache holds of rows in 32 bits, as values in 32 bits."""
    if store not in (I8, E4M3):
        return x.to(store).float()
    most = x.abs().amax(-1, keepdim=True)
    big = torch.full_like(most, 127.0 if store == I8 else 448.0)  # a tensor: torch divides by a number by way of its reciprocal
    code = torch.where(most == 0, 0.0, x * (big / most))
    code = code.round().clamp(-127, 127) if store == I8 else code.clamp(-448, 448).to(E4M3).float()
    return code * (most / big)


CACHE = [
    # lengths, heads, dim, page, type, store, indices
    ([1], 1, 1, 1, F32, F32, torch.int32),
    ([5, 0, 17, 3], 2, 128, 16, BF16, BF16, torch.int32),
    ([5, 0, 17, 3], 3, 128, 16, BF16, I8, torch.int64),
    ([40], 8, 128, 64, F16, E4M3, torch.int32),
    ([9, 30], 5, 80, 24, F16, I8, torch.int32),
    ([9, 30], 2, 72, 7, F32, E4M3, torch.int32),
    ([9, 30], 2, 37, 3, F32, I8, torch.int32),
    ([3, 4], 4, 256, 8, F32, F32, torch.int64),
    ([3, 4], 4, 256, 8, BF16, E4M3, torch.int32),
    ([100], 1, 64, 32, F16, F16, torch.int32),
    ([100], 1, 20, 32, BF16, I8, torch.int32),
    ([257, 1, 64], 4, 96, 16, F32, I8, torch.int32),
]


def make_cache(A, case, extra=2):
    lens, heads, dim, page, dtype, store, idx = case
    each = [-(-n // page) for n in lens]
    pages = sum(each) + extra
    cache = A.PagedCache.empty(pages, heads, page, dim, store)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0xff)  # not a number, but for int8
    for t in (cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(math.nan)
    pos, crd = lists(each, pages, 7, idx)
    return cache, pos, crd


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("c", CACHE, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_append_and_read(A, c, strided):
    """Bit for bit: the codes are products and roundings in 32 bits."""
    lens, heads, dim, page, dtype, store, idx = c
    cache, pos, crd = make_cache(A, c)
    before = [t.clone() for t in (cache.k, cache.v)]
    row, place = tokens_of(lens, idx)
    x = normal(1, len(row), 2 * heads, dim + (1 if strided else 0)).to(dtype)
    if len(row) > 2:
        x[1] = 0                    # a row of zeros
        x[2, 0] *= 1e-3
        x[2, :, 0] = 100.0
    k, v = x[:, :heads, :dim], x[:, heads:, :dim]
    order = torch.from_numpy(np.random.default_rng(2).permutation(len(row))).to(DEV)
    cache.append(k[order], v[order], pos, crd, row[order], place[order])
    for out in (F32, dtype):
        got = cache.read(pos, crd, row, place, dtype=out)
        for y, z in zip(got, (k, v)):
            assert y.dtype == out and torch.equal(y, quantised(z.float(), store).to(out))
    # nothing else was written
    page_of = crd.long()[pos.long()[row.long()] + place.long() // page]
    for now, then in zip((cache.k, cache.v), before):
        now, then = now.view(torch.uint8).clone(), then.view(torch.uint8).clone()
        now[page_of, :, place.long() % page] = then[page_of, :, place.long() % page]
        assert torch.equal(now, then)


@pytest.mark.parametrize("c", [c for c in CACHE if c[2] % 2 == 0], ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_append_norm_rope(A, c):
    """The queries are those of qk_norm_rope; the keys are off by half a step of their code, and by the rounding of what is quantised."""
    lens, heads, dim, page, dtype, store, idx = c
    cache, pos, crd = make_cache(A, c)
    row, place = tokens_of(lens, idx)
    x = normal(1, len(row), 5 * heads, dim).to(dtype)
    q, k, v = x[:, :3 * heads], x[:, 3 * heads:4 * heads], x[:, 4 * heads:]
    w = (1 + 0.3 * normal(2, 2, dim)).to(dtype)
    cos, sin = tables(300, dim)
    got_q = cache.append_norm_rope(q, k, v, w[0], w[1], cos, sin, pos, crd, row, place, eps=1e-5, interleaved=True)
    want_q, want_k = A.qk_norm_rope(q, k, w[0], w[1], cos, sin, place, eps=1e-5, interleaved=True)
    assert torch.equal(got_q, want_q)
    got_k, got_v = cache.read(pos, crd, row, place, dtype=F32)
    assert torch.equal(got_v, quantised(v.float(), store))
    if store not in (I8, E4M3):
        assert torch.equal(got_k, want_k.float())
        return
    exact = forward64(k, w[1], cos, sin, place.long(), 1e-5, True)
    most, off = exact.abs().amax(-1, keepdim=True), (dim + 32) * E * partners(exact, dim, True)
    step = most / 127 * 0.5 if store == I8 else torch.maximum(exact.abs() * 2.0 ** -4, most / 448 * 2.0 ** -10)
    assert bool(((got_k.double() - exact).abs() <= step * (1 + 1e-4) + off + 2 * E * exact.abs()).all())


@pytest.mark.parametrize("store", [BF16, I8])
def test_cache_ignores_what_the_lists_do_not_cover(A, store):
    c = ([20, 20], 2, 64, 8, BF16, store, torch.int32)
    cache, pos, crd = make_cache(A, c, extra=3)
    before = [t.clone() for t in (cache.k, cache.v)]
    row = torch.tensor([0, 0, -1, 2, 1, 1, 0], device=DEV, dtype=torch.int32)
    place = torch.tensor([24, -1, 0, 0, 2 ** 31 - 1, 8, 8], device=DEV, dtype=torch.int32)
    bad = crd.clone()
    bad[1], bad[4] = -3, cache.pages
    x = normal(3, 7, 2, 64).bfloat16()
    cache.append(x, x, pos, bad, row, place)
    cos, sin = tables(4, 64)
    w = torch.ones(64, device=DEV)
    cache.append_norm_rope(x, x, x, w, w, cos, sin, pos, crd, torch.zeros(7, device=DEV, dtype=torch.int32),
                           torch.where(place < 4, 50 - place, place))  # padding: beyond the tables
    assert torch.equal(cache.k.view(torch.uint8), before[0].view(torch.uint8))
    assert torch.equal(cache.v.view(torch.uint8), before[1].view(torch.uint8))
    for y in cache.read(pos, bad, row, place):
        assert y.dtype == BF16 and float(y.abs().max()) == 0
    none = torch.zeros(0, device=DEV, dtype=torch.int32)
    assert cache.read(pos, crd, none, none)[0].shape == (0, 2, 64)
    cache.append(x[:0], x[:0], pos, crd, none, none)


@pytest.mark.parametrize("store", [I8, E4M3])
@pytest.mark.parametrize("dim", [64, 20])
def test_rows_that_are_not_finite_read_as_nan(A, store, dim):
    c = ([4], 1, dim, 4, F32, store, torch.int32)
    cache, pos, crd = make_cache(A, c)
    row, place = tokens_of([4])
    x = normal(3, 4, 1, dim).float()
    x[0, 0, 3], x[2, 0, 5] = math.inf, math.nan
    cache.append(x, x, pos, crd, row, place)
    for y in cache.read(pos, crd, row, place, dtype=F32):
        assert bool(y[[0, 2]].isnan().all()) and bool(y[[1, 3]].isfinite().all())


# ---- attention --------------------------------------------------------------

ATTEND = [
    # lengths, q heads, kv heads, dim, page, type, store, window
    ([1], 1, 1, 128, 16, BF16, BF16, 0),
    ([0], 4, 2, 128, 16, BF16, BF16, 0),
    ([0, 3, 0, 65, 0], 8, 2, 128, 16, BF16, I8, 0),
    ([2, 16, 17, 63, 64, 65], 4, 4, 128, 16, BF16, BF16, 0),
    ([300, 1, 90], 16, 2, 128, 64, F16, F16, 0),
    ([300, 1, 90], 16, 2, 128, 64, F16, E4M3, 0),
    ([1000, 1025], 32, 2, 128, 24, BF16, E4M3, 0),         # 16 query heads a key head
    ([130], 17, 1, 128, 1, BF16, BF16, 0),                 # 17
    ([130, 7], 40, 1, 64, 16, BF16, I8, 0),                # 40
    ([200, 511], 9, 3, 64, 8, F16, F16, 0),
    ([200, 511], 18, 2, 64, 128, F16, I8, 0),              # 9
    ([77, 500], 6, 2, 256, 16, BF16, BF16, 0),
    ([77, 500], 20, 2, 256, 16, F16, E4M3, 0),
    ([77, 500], 6, 2, 256, 16, BF16, I8, 0),
    ([77, 500], 6, 2, 96, 24, BF16, BF16, 0),
    ([77, 500], 6, 2, 80, 16, F16, E4M3, 0),
    ([77, 500], 6, 2, 112, 16, BF16, I8, 0),
    ([77, 500], 6, 2, 192, 16, BF16, BF16, 0),
    ([77, 500], 6, 2, 72, 16, F16, F16, 0),
    ([77, 500], 6, 2, 72, 16, BF16, I8, 0),                # no whole 16 bytes of codes
    ([77, 500], 6, 2, 36, 16, BF16, E4M3, 0),
    ([77, 500], 3, 3, 32, 16, BF16, E4M3, 0),
    ([77, 500], 3, 3, 16, 16, F16, I8, 0),
    ([77, 500], 3, 3, 8, 16, F16, F16, 0),
    ([50, 33], 3, 1, 5, 3, BF16, BF16, 0),
    ([50, 33], 3, 1, 1, 3, F32, F32, 0),
    ([500, 333], 8, 2, 128, 16, F32, F32, 0),
    ([500, 333], 8, 8, 72, 24, F32, F32, 0),
    ([500, 333], 24, 2, 64, 16, F32, I8, 0),
    ([500, 333], 5, 1, 256, 16, F32, E4M3, 0),
    ([500, 33, 0, 128, 129], 8, 2, 128, 16, BF16, BF16, 128),
    ([500, 33, 0, 128, 129], 8, 2, 64, 16, F16, E4M3, 1),
    ([500, 33, 0, 128, 129], 8, 2, 64, 16, F32, F32, 100),
    ([500, 3000], 8, 2, 128, 32, BF16, I8, 777),
    ([70001], 8, 1, 128, 64, BF16, BF16, 0),               # one request over all blocks
    ([70001, 3], 4, 2, 64, 16, F16, I8, 0),
    ([9000, 1], 4, 1, 40, 16, F32, F32, 0),
    (list(range(0, 400, 3)), 4, 2, 128, 16, BF16, BF16, 0),   # 134 ragged requests
    ([40] * 700, 2, 1, 64, 16, BF16, E4M3, 0),
    # 32 bits: eight, four and one query heads a unit, wide and narrow heads, pages that split a group of keys
    ([300, 0, 41], 8, 1, 64, 16, F32, F32, 0),
    ([300, 0, 41], 5, 1, 128, 12, F32, F32, 0),
    ([300, 0, 41], 11, 1, 256, 16, F32, F32, 0),
    ([300, 0, 41], 9, 3, 256, 8, F32, F32, 50),
    ([300, 0, 41], 2, 2, 256, 1, F32, F32, 0),
    ([300, 0, 41], 2, 2, 32, 24, F32, F32, 33),
    ([2500], 20, 2, 100, 64, F32, F32, 0),
    ([70001, 5], 2, 2, 128, 16, F32, F32, 0),
    ([300, 0, 41], 20, 1, 128, 16, F32, E4M3, 0),
    ([300, 0, 41], 20, 2, 64, 12, F32, I8, 100),
    ([300, 700], 3, 1, 256, 16, F32, I8, 0),
    ([5000], 4, 4, 72, 16, F32, I8, 0),
    # rows of whole 8 bytes, and of less
    ([300, 0, 41], 4, 2, 36, 16, F16, F16, 0),
    ([300, 0, 41], 4, 2, 100, 12, BF16, BF16, 40),
    ([300, 0, 41], 20, 2, 132, 16, BF16, BF16, 0),
    ([300, 0, 41], 4, 2, 40, 5, F16, E4M3, 0),
    ([300, 0, 41], 4, 2, 200, 16, BF16, I8, 0),
    ([300, 0, 41], 4, 2, 34, 16, F16, F16, 0),
    ([300, 0, 41], 4, 2, 66, 16, F32, F32, 0),
    # windows whose first key is no multiple of 16, of whole and of cut units
    ([6000, 17, 100], 8, 2, 128, 16, BF16, BF16, 1001),
    ([6000, 17, 100], 32, 2, 128, 48, F16, I8, 1001),
    ([60000, 59999], 2, 1, 64, 128, F16, E4M3, 50007),
    # many requests: more than a thread each, and many that are short
    ([3] * 300 + [900, 0, 5] + [1] * 40, 8, 2, 128, 16, BF16, I8, 0),
    ([17] * 500, 4, 4, 64, 16, F32, F32, 0),
]


def fill(cache, pos, crd, lens, seed, dtype):
    """Writes what the requests hold and returns it in 64 bits: (k, v) [tokens, heads, dim] of each request.  Slots that hold
    nothing keep NaN."""
    got = []
    row, place = tokens_of(lens, pos.dtype)
    k, v = normal(seed, len(row), cache.heads, cache.dim).to(dtype), normal(seed + 1, len(row), cache.heads, cache.dim).to(dtype)
    cache.append(k, v, pos, crd, row, place)
    store = cache.k.dtype
    k, v = quantised(k.float(), store).double(), quantised(v.float(), store).double()
    at = 0
    for n in lens:
        got.append((k[at:at + n], v[at:at + n]))
        at += n
    return got


def attend64(q, held, scale, window):
    """out, lse, and the bounds of both but for the rounding of `out`."""
    group = q.shape[1] // held[0][0].shape[1] if held else 1
    outs = []
    for b, (k, v) in enumerate(held):
        if window:
            k, v = k[-window:], v[-window:]
        n, dim = len(k), q.shape[2]
        if n == 0:
            outs.append((torch.zeros(q.shape[1:], device=DEV, dtype=torch.float64), torch.full((q.shape[1],), -math.inf, device=DEV, dtype=torch.float64),
                         torch.zeros(q.shape[1:], device=DEV, dtype=torch.float64), torch.zeros(q.shape[1], device=DEV, dtype=torch.float64)))
            continue
        k, v = (x.repeat_interleave(group, 1) for x in (k, v))
        s = torch.einsum("hd,nhd->hn", q[b].double(), k) * scale
        lse = torch.logsumexp(s, -1)
        p = (s - lse[:, None]).exp()
        size = torch.einsum("hd,nhd->hn", q[b].double().abs(), k.abs()) * abs(scale)
        ds = 4 * (dim + 8) * E * size.amax(-1) + 8 * E * (1 + s.abs().amax(-1))
        of_weights = 2 * ds + (n + 64) * 4 * E + WEIGHT[q.dtype]
        outs.append((torch.einsum("hn,nhd->hd", p, v), lse, of_weights[:, None] * torch.einsum("hn,nhd->hd", p, v.abs()), ds + (n + 64) * E + 4 * E * lse.abs()))
    return [torch.stack(x) for x in zip(*outs)]


def holds(q, got, want):
    out, lse = got
    exact, exact_lse, bound, bound_lse = want
    assert out.dtype == q.dtype and lse.dtype == F32
    assert bool(((out.double() - exact).abs() <= bound + U[q.dtype] * exact.abs() + TINY[q.dtype]).all())
    some = exact_lse.isfinite()
    assert torch.equal(lse[~some].double(), exact_lse[~some])
    assert bool(((lse.double() - exact_lse).abs()[some] <= bound_lse[some]).all())


@pytest.mark.parametrize("c", ATTEND, ids=lambda c: "-".join((str(x) if len(str(x)) < 30 else "%d_requests" % len(x)).replace("torch.", "") for x in c))
def test_attend(A, c):
    lens, hq, hkv, dim, page, dtype, store, window = c
    idx = torch.int64 if len(lens) == 2 else torch.int32
    cache, pos, crd = make_cache(A, (lens, hkv, dim, page, dtype, store, idx))
    held = fill(cache, pos, crd, lens, 11, dtype)
    q = (2 * normal(5, len(lens), hq, dim)).to(dtype)
    length = torch.tensor(lens, device=DEV, dtype=idx)
    got = A.paged_attention(q, cache, pos, crd, length, window=window, return_lse=True)
    holds(q, got, attend64(q, held, dim ** -0.5, window))
    again = A.paged_attention(q, cache, pos, crd, length, window=window, return_lse=True)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert torch.equal(got[0], A.paged_attention(q, cache, pos, crd, length, window=window))


@pytest.mark.parametrize("strided", ["view", "odd", "heads first"])
@pytest.mark.parametrize("dtype,store,dim", [(BF16, BF16, 128), (F16, I8, 64), (F32, F32, 40), (BF16, E4M3, 256)])
def test_attend_strides(A, dtype, store, dim, strided):
    lens = [100, 37, 250]
    cache, pos, crd = make_cache(A, (lens, 2, dim, 16, dtype, store, torch.int32))
    held = fill(cache, pos, crd, lens, 11, dtype)
    x = normal(5, 3, 12, dim + (1 if strided == "odd" else 0)).to(dtype)
    if strided == "heads first":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    q = x[:, 2:10, :dim]
    length = torch.tensor(lens, device=DEV, dtype=torch.int32)
    holds(q, A.paged_attention(q, cache, pos, crd, length, scale=0.3, return_lse=True), attend64(q, held, 0.3, 0))


@pytest.mark.parametrize("dtype,store,dim", [(BF16, BF16, 128), (BF16, I8, 128), (F16, E4M3, 64), (F32, F32, 72)])
def test_attend_large_scores_and_values(A, dtype, store, dim):
    """Scores of some hundreds, later ones much larger than earlier ones; values and scales over many orders of magnitude."""
    lens = [3000, 200]
    cache, pos, crd = make_cache(A, (lens, 1, dim, 16, dtype, store, torch.int32))
    row, place = tokens_of(lens)
    grow = 2.0 ** (-12 + 14 * place.double() / 3000)[:, None, None]
    k, v = (normal(1, len(row), 1, dim) * 0.5 * grow.sqrt()).to(dtype), (normal(2, len(row), 1, dim) / grow).to(dtype)
    cache.append(k, v, pos, crd, row, place)
    held = [tuple(quantised(x[a:b].float(), store).double() for x in (k, v)) for a, b in ((0, 3000), (3000, 3200))]
    q = (30 * normal(5, 2, 4, dim)).to(dtype)
    length = torch.tensor(lens, device=DEV, dtype=torch.int32)
    holds(q, A.paged_attention(q, cache, pos, crd, length, return_lse=True), attend64(q, held, dim ** -0.5, 0))


@pytest.mark.parametrize("dtype,store,dim", [(BF16, BF16, 128), (BF16, I8, 64), (F32, F32, 24)])
def test_attend_small_queries_and_zero_rows(A, dtype, store, dim):
    """Queries of 1e-30 weigh all keys alike; a cache of zeros gives zeros."""
    lens = [130]
    cache, pos, crd = make_cache(A, (lens, 1, dim, 16, dtype, store, torch.int32))
    held = fill(cache, pos, crd, lens, 11, dtype)
    length = torch.tensor(lens, device=DEV, dtype=torch.int32)
    q = (1e-30 * normal(5, 1, 2, dim)).to(dtype)
    holds(q, A.paged_attention(q, cache, pos, crd, length, return_lse=True), attend64(q, held, dim ** -0.5, 0))
    row, place = tokens_of(lens)
    zero = torch.zeros(130, 1, dim, device=DEV, dtype=dtype)
    cache.append(zero, zero, pos, crd, row, place)
    out, lse = A.paged_attention(q, cache, pos, crd, length, return_lse=True)
    assert float(out.abs().max()) == 0 and torch.allclose(lse, torch.full_like(lse, math.log(130)), rtol=1e-6)


@pytest.mark.parametrize("dtype,store,dim", [(BF16, BF16, 128), (F16, E4M3, 64), (F32, F32, 20)])
def test_attend_bad_lists(A, dtype, store, dim):
    """A length beyond the listed pages ends with them; pages that do not exist read as zeros."""
    lens = [40, 32, 16]
    cache, pos, crd = make_cache(A, (lens, 2, dim, 8, dtype, store, torch.int32))
    held = fill(cache, pos, crd, lens, 11, dtype)
    crd[6] = cache.pages + 5   # places 8 to 15 of request 1
    crd[10] = -1               # 8 to 15 of request 2
    for r in (1, 2):
        for x in held[r]:
            x[8:16] = 0
    q = normal(5, 3, 4, dim).to(dtype)
    length = torch.tensor([1000, 32, 16], device=DEV, dtype=torch.int32)
    holds(q, A.paged_attention(q, cache, pos, crd, length, return_lse=True), attend64(q, held, dim ** -0.5, 0))
    assert float(A.paged_attention(q, cache, pos, crd, -length).abs().max()) == 0


@pytest.mark.parametrize("dtype,store,dim", [(BF16, BF16, 128), (BF16, I8, 128), (F32, F32, 24)])
def test_attend_not_finite(A, dtype, store, dim):
    """A NaN among a request's keys is seen by the heads that read it and by no others."""
    lens = [100, 100]
    cache, pos, crd = make_cache(A, (lens, 2, dim, 16, dtype, store, torch.int32))
    row, place = tokens_of(lens)
    k, v = normal(1, 200, 2, dim).to(dtype), normal(2, 200, 2, dim).to(dtype)
    k[70, 1, 3] = math.nan
    cache.append(k, v, pos, crd, row, place)
    q = normal(5, 2, 4, dim).to(dtype)
    out, lse = A.paged_attention(q, cache, pos, crd, torch.tensor(lens, device=DEV, dtype=torch.int32), return_lse=True)
    assert bool(out[0, 2:].isnan().all()) and bool(lse[0, 2:].isnan().all())
    assert bool(out[0, :2].isfinite().all()) and bool(out[1].isfinite().all()) and bool(lse[1].isfinite().all())


def test_attend_parts_join_by_lse(A):
    """Halves of a context joined by their lse are the whole."""
    cache, pos, crd = make_cache(A, ([512], 2, 128, 64, F32, F32, torch.int32))
    fill(cache, pos, crd, [512], 11, F32)
    q = normal(5, 1, 8, 128).float()
    whole, lse = A.paged_attention(q, cache, pos, crd, torch.tensor([512], device=DEV, dtype=torch.int32), return_lse=True)
    parts = [A.paged_attention(q, cache, torch.tensor([0, 4], device=DEV, dtype=torch.int32), crd[4 * i:4 * i + 4].contiguous(),
                               torch.tensor([256], device=DEV, dtype=torch.int32), return_lse=True) for i in range(2)]
    w = torch.softmax(torch.stack([p[1] for p in parts]), 0)
    assert torch.allclose(whole, sum(p[0] * w[i][..., None] for i, p in enumerate(parts)), rtol=1e-4, atol=1e-5)
    assert torch.allclose(lse, torch.logsumexp(torch.stack([p[1] for p in parts]), 0), rtol=1e-5)


def test_step_on_another_stream_and_in_a_graph(A):
    """Write and attend in order on a stream of their own, and replayed from a captured graph with other inputs."""
    lens = [33, 64, 5, 200]
    c = (lens, 2, 128, 16, BF16, BF16, torch.int32)
    cache, pos, crd = make_cache(A, c)
    held = fill(cache, pos, crd, lens, 11, BF16)
    length = torch.tensor(lens, device=DEV, dtype=torch.int32)
    place, row = length - 1, torch.arange(4, device=DEV, dtype=torch.int32)
    w, (cos, sin) = torch.ones(128, device=DEV), tables(200, 128)
    qkv = normal(1, 4, 12, 128).bfloat16()

    def step():
        q = cache.append_norm_rope(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], w, w, cos, sin, pos, crd, row, place)
        return q, A.paged_attention(q, cache, pos, crd, length, return_lse=True)

    def check(q, got):
        k = A.qk_norm_rope(qkv[:, :8], qkv[:, 8:10], w, w, cos, sin, place)[1].double()
        now = [(torch.cat([h[0][:-1], k[b][None]]), torch.cat([h[1][:-1], qkv[b, 10:].double()[None]])) for b, h in enumerate(held)]
        holds(q, got, attend64(q, now, 128 ** -0.5, 0))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    check(*first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (2, 3):
        qkv.copy_(normal(seed, 4, 12, 128))
        graph.replay()
        torch.cuda.synchronize()
        check(*got)


def test_attend_rows_beyond_32_bits(A):
    """Elements of the cache whose offset does not fit 32 bits."""
    heads, page, dim = 2, 64, 128
    pages = 2 ** 31 // (heads * page * dim) + 40   # 4.3 GB each of keys and values
    cache = A.PagedCache(*(torch.zeros(pages, heads, page, dim, device=DEV, dtype=BF16) for _ in range(2)))
    lens = [130, 70]
    pos = torch.tensor([0, 3, 5], device=DEV, dtype=torch.int32)
    crd = torch.tensor([pages - 1, 0, pages - 7, pages - 30, pages - 2], device=DEV, dtype=torch.int32)
    held = fill(cache, pos, crd, lens, 11, BF16)
    row, place = tokens_of(lens)
    got = cache.read(pos, crd, row, place, dtype=BF16)
    assert torch.equal(got[0].double(), torch.cat([h[0] for h in held])) and torch.equal(got[1].double(), torch.cat([h[1] for h in held]))
    q = normal(5, 2, 8, dim).bfloat16()
    holds(q, A.paged_attention(q, cache, pos, crd, torch.tensor(lens, device=DEV, dtype=torch.int32), return_lse=True), attend64(q, held, dim ** -0.5, 0))


# ---- what the calls refuse ----------------------------------------------------


@pytest.mark.parametrize("error,change", [
    (TypeError, {"q": None}), (ValueError, {"q": lambda t: t[0]}), (TypeError, {"q": lambda t: t.double()}), (TypeError, {"q": lambda t: t.cpu()}),
    (TypeError, {"q": lambda t: t.half()}), (TypeError, {"q": lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)}),
    (TypeError, {"k": lambda t: t.half()}), (ValueError, {"k": lambda t: t[:2]}), (ValueError, {"v": lambda t: t[:, :1]}), (ValueError, {"k": lambda t: t[..., :32]}),
    (ValueError, {"q_weight": lambda t: t[:32]}), (TypeError, {"k_weight": lambda t: t.double()}), (TypeError, {"q_weight": None}),
    (ValueError, {"sin": lambda t: t[:5]}), (TypeError, {"cos": lambda t: t.half()}), (ValueError, {"cos": lambda t: t.repeat(1, 2), "sin": lambda t: t.repeat(1, 2)}),
    (TypeError, {"place": lambda t: t.float()}), (ValueError, {"place": lambda t: t[:2]}), (TypeError, {"row": lambda t: t.float()}), (ValueError, {"row": lambda t: t[:2]}),
    (TypeError, {"crd": lambda t: t.long()}), (TypeError, {"pos": None}), (ValueError, {"pos": lambda t: t[:0]}), (TypeError, {"place": lambda t: t[::2].repeat_interleave(2)[::2]}),
])
def test_append_norm_rope_raises(A, error, change):
    cache, pos, crd = make_cache(A, ([8, 8], 2, 64, 4, BF16, I8, torch.int32))
    cos, sin = tables(8, 64)
    x = normal(1, 4, 8, 64).bfloat16()
    i32 = dict(device=DEV, dtype=torch.int32)
    a = dict(q=x[:, :4], k=x[:, 4:6], v=x[:, 6:], q_weight=torch.ones(64, device=DEV), k_weight=torch.ones(64, device=DEV), cos=cos, sin=sin, pos=pos, crd=crd,
             row=torch.tensor([0, 0, 1, 1], **i32), place=torch.tensor([0, 1, 0, 1], **i32))
    cache.append_norm_rope(**a)
    before = cache.k.clone()
    for name, f in change.items():
        a[name] = f(a[name]) if f else None
    with pytest.raises(error):
        cache.append_norm_rope(**a)
    if not {"pos", "crd", "row", "v"} & set(change):
        b = {n: a[n] for n in ("q", "k", "q_weight", "k_weight", "cos", "sin", "place")}
        with pytest.raises(error):
            A.qk_norm_rope(**b)
        with pytest.raises(error):
            A.qk_norm_rope_backward(a["q"], a["k"], **b)
    if {"k", "v", "row", "place", "pos", "crd"} & set(change):
        with pytest.raises(error):
            cache.append(a["k"], a["v"], pos=a["pos"], crd=a["crd"], row=a["row"], place=a["place"])
    if {"row", "place", "pos", "crd"} & set(change):
        with pytest.raises(error):
            cache.read(a["pos"], a["crd"], a["row"], a["place"])
    torch.cuda.synchronize()
    assert torch.equal(cache.k, before)


@pytest.mark.parametrize("error,change", [
    (TypeError, {"q": None}), (ValueError, {"q": lambda t: t[0]}), (TypeError, {"q": lambda t: t.double()}), (TypeError, {"q": lambda t: t.cpu()}),
    (ValueError, {"q": lambda t: t[..., :32]}), (ValueError, {"length": lambda t: t[:1]}), (TypeError, {"length": lambda t: t.long()}),
    (TypeError, {"crd": lambda t: t.float()}), (ValueError, {"pos": lambda t: t[:0]}),
])
def test_attention_raises(A, error, change):
    from lapis_b200._lib import LapisError
    cache, pos, crd = make_cache(A, ([8, 8], 2, 64, 4, BF16, I8, torch.int32))
    a = dict(q=normal(1, 2, 4, 64).bfloat16(), pos=pos, crd=crd, length=torch.tensor([3, 5], device=DEV, dtype=torch.int32))
    for name, f in change.items():
        a[name] = f(a[name]) if f else None
    with pytest.raises(error):
        A.paged_attention(cache=cache, **a)
    with pytest.raises(TypeError):
        cache.read(pos, crd, pos[:2], pos[:2], dtype=torch.float64)
    with pytest.raises(LapisError):  # three query heads over two
        A.paged_attention(normal(1, 2, 3, 64).bfloat16(), cache, pos, crd, torch.tensor([3, 5], device=DEV, dtype=torch.int32))
    with pytest.raises(LapisError):  # a list too few
        A.paged_attention(normal(1, 2, 4, 64).bfloat16(), cache, pos[:2], crd, torch.tensor([3, 5], device=DEV, dtype=torch.int32))
    with pytest.raises(LapisError):
        A.paged_attention(normal(1, 2, 4, 64).bfloat16(), cache, pos, crd, torch.tensor([3, 5], device=DEV, dtype=torch.int32), scale=math.inf)


@pytest.mark.parametrize("store", [BF16, I8, F32])
def test_cache_without_pages(A, store):
    """No page at all: zeros, whatever the lists say."""
    dtype = F32 if store == F32 else BF16
    cache = A.PagedCache.empty(0, 2, 16, 64, store)
    pos, crd = torch.tensor([0, 2, 2], device=DEV, dtype=torch.int32), torch.tensor([0, 5], device=DEV, dtype=torch.int32)
    row, place = torch.tensor([0, 1], device=DEV, dtype=torch.int32), torch.tensor([3, 0], device=DEV, dtype=torch.int32)
    x = normal(1, 2, 2, 64).to(dtype)
    cache.append(x, x, pos, crd, row, place)
    assert float(cache.read(pos, crd, row, place, dtype=F32)[0].abs().max()) == 0
    out, lse = A.paged_attention(normal(1, 2, 4, 64).to(dtype), cache, pos, crd, torch.tensor([20, 0], device=DEV, dtype=torch.int32), return_lse=True)
    assert float(out.abs().max()) == 0 and torch.allclose(lse[0], torch.full((4,), math.log(20), device=DEV), rtol=1e-6) and bool((lse[1] == -math.inf).all())
