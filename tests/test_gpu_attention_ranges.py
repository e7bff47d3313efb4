"""Attention over quantised and 16-bit caches where scores, values and scales lie far apart: against 64 bits, with the bounds of
test_gpu_attention.py where none is derived here."""
import math

import pytest
import torch

from tests.test_gpu_attention import BF16, DEV, E, E4M3, F16, F32, I8, TINY, U, WEIGHT, attend64, holds, make_cache, normal, quantised, tokens_of

pytestmark = pytest.mark.gpu

CODES = [(BF16, I8, 128), (BF16, E4M3, 64), (F16, I8, 64), (F16, E4M3, 256), (F32, I8, 128), (F32, E4M3, 64), (F32, I8, 20)]


@pytest.fixture(scope="module")
def A():
    from lapis_b200 import attention
    return attention


def length_of(lens):
    return torch.tensor(lens, device=DEV, dtype=torch.int32)


# ---- scores of 10^8 ----------------------------------------------------------


@pytest.mark.parametrize("heads", [2, 12])
@pytest.mark.parametrize("lens", [[40], [3000, 70]])
@pytest.mark.parametrize("dtype,store,dim", [(F16, F16, 64), (F16, F16, 256), (F16, I8, 64), (F16, E4M3, 128), (BF16, I8, 64), (BF16, BF16, 64), (F32, I8, 64),
                                             (F32, F32, 64)])
def test_one_key_far_above_all_others(A, dtype, store, dim, lens, heads):
    """Its weight is one and all others are zero: out is its value, off by the rounding of its weight in front of the product and by 8
    units of 32 bits; lse is its score, a sum of `dim` products in 32 bits."""
    cache, pos, crd = make_cache(A, (lens, 1, dim, 16, dtype, store, torch.int32))
    row, place = tokens_of(lens)
    k, v = normal(1, len(row), 1, dim).to(dtype), normal(2, len(row), 1, dim).to(dtype)
    at = [17, lens[0] + 33][:len(lens)]
    top = 4096.0 * 8 / math.sqrt(dim)
    k[at] = top
    cache.append(k, v, pos, crd, row, place)
    q = torch.full((len(lens), heads, dim), 4096.0, device=DEV, dtype=dtype)
    q[:, 1::2] *= 1.25
    out, lse = A.paged_attention(q, cache, pos, crd, length_of(lens), return_lse=True)
    held, k = quantised(v.float(), store).double(), quantised(k.float(), store).double()
    for b, j in enumerate(at):
        want = held[j].expand(heads, dim)
        assert bool(((out[b].double() - want).abs() <= (U[dtype] + WEIGHT[dtype] + 2.0 ** -21) * want.abs() + 2.0 ** -24).all())
        score = (q[b].double() * k[j].double()).sum(-1) * dim ** -0.5
        assert bool(((lse[b].double() - score).abs() <= 4 * (dim + 8) * 2.0 ** -24 * score.abs()).all())


# ---- values of 10^36 ---------------------------------------------------------


@pytest.mark.parametrize("lens", [[30, 5], [3000]])
@pytest.mark.parametrize("dtype,store,dim", [c for c in CODES if c[0] != F16])
def test_values_near_the_largest_number(A, dtype, store, dim, lens):
    """Sums of the weights' products with values of up to 10^34 for 3000 tokens, 10^36 for 30, are numbers of 32 bits."""
    cache, pos, crd = make_cache(A, (lens, 1, dim, 16, dtype, store, torch.int32))
    row, place = tokens_of(lens)
    k, v = normal(1, len(row), 1, dim).to(dtype), (normal(2, len(row), 1, dim) * (2e36 if lens[0] == 30 else 3e34)).to(dtype)
    cache.append(k, v, pos, crd, row, place)
    held, at = [], 0
    for n in lens:
        held.append(tuple(quantised(x[at:at + n].float(), store).double() for x in (k, v)))
        at += n
    q = normal(5, len(lens), 4, dim).to(dtype)
    holds(q, A.paged_attention(q, cache, pos, crd, length_of(lens), return_lse=True), attend64(q, held, dim ** -0.5, 0))


# ---- scales of a caller's own cache ------------------------------------------


@pytest.mark.parametrize("signs", ["mixed", "negative"])
@pytest.mark.parametrize("dtype,store,dim", CODES)
def test_negative_scales(A, dtype, store, dim, signs):
    lens = [130, 7]
    cache, pos, crd = make_cache(A, (lens, 2, dim, 16, dtype, store, torch.int32))
    row, place = tokens_of(lens)
    k, v = normal(1, len(row), 2, dim).to(dtype), normal(2, len(row), 2, dim).to(dtype)
    cache.append(k, v, pos, crd, row, place)
    sign = torch.where(normal(3, 2, *cache.k_scale.shape) < 0, -1.0, 1.0) if signs == "mixed" else torch.full((2, *cache.k_scale.shape), -1.0, device=DEV)
    cache.k_scale *= sign[0]
    cache.v_scale *= sign[1]
    k, v = cache.read(pos, crd, row, place, dtype=F32)
    held = [(k[:130].double(), v[:130].double()), (k[130:].double(), v[130:].double())]
    q = normal(5, 2, 6, dim).to(dtype)
    holds(q, A.paged_attention(q, cache, pos, crd, length_of(lens), return_lse=True), attend64(q, held, dim ** -0.5, 0))


# ---- scales far apart ----------------------------------------------------------


def held_to(q, got, held, scale):
    """As holds(); what fp16 leaves of weight * scale of a key is also off by 2^-38 of the largest one of its head, which shows where the codes
    that count most are zeros."""
    out, lse, bound, bound_lse = attend64(q, held, scale, 0)
    for b, (k, v) in enumerate(held):
        p = (torch.einsum("hd,nd->hn", q[b].double(), k[:, 0]) * scale - lse[b][:, None]).exp()
        most = v[:, 0].abs().amax(-1)  # 127 (448) times the scale
        bound[b] += 2.0 ** -38 * (p * most).amax(-1)[:, None] * (v[:, 0].abs() / most[:, None]).sum(0)
    holds(q, got, (out, lse, bound, bound_lse))


def apart(A, dtype, store, dim, lens, ratio, first, values=1.0):
    """Requests of which one token's values are `ratio` times the others'; heads 0, 2, ... give it a weight of about e^-60 of theirs,
    the others nearly all weight."""
    cache, pos, crd = make_cache(A, (lens, 1, dim, 16, dtype, store, torch.int32))
    row, place = tokens_of(lens)
    q = (1 + 0.1 * normal(5, len(lens), 4, dim)) * torch.tensor([1.0, -1.0, 1.0, -1.0], device=DEV)[:, None]
    k, v = 0.3 * normal(1, len(row), 1, dim), values * normal(2, len(row), 1, dim)
    start = 0
    for n in lens:
        j = start + (1 if first else n - 2)
        k[j] = -60 / math.sqrt(dim)
        v[j] *= ratio
        start += n
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    cache.append(k, v, pos, crd, row, place)
    held, start = [], 0
    for n in lens:
        held.append(tuple(quantised(x[start:start + n].float(), store).double() for x in (k, v)))
        start += n
    held_to(q, A.paged_attention(q, cache, pos, crd, length_of(lens), return_lse=True), held, dim ** -0.5)


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("lens", [[100], [3000, 33]])
@pytest.mark.parametrize("power", [18, 24, 32, 40, 60])
@pytest.mark.parametrize("dtype,store,dim", [c for c in CODES if c[0] != F16])
def test_value_scales_far_apart(A, dtype, store, dim, power, lens, first):
    apart(A, dtype, store, dim, lens, 2.0 ** power, first)


@pytest.mark.parametrize("dtype,store,dim", [(F16, I8, 64), (F16, E4M3, 256)])
def test_value_scales_far_apart_fp16(A, dtype, store, dim):
    apart(A, dtype, store, dim, [100, 700], 2.0 ** 20, False, 2.0 ** -8)


@pytest.mark.parametrize("values", [1e-30, 1e-34, 1e30])
@pytest.mark.parametrize("dtype,store,dim", [c for c in CODES if c[0] != F16])
def test_small_and_large_values(A, dtype, store, dim, values):
    apart(A, dtype, store, dim, [100, 700], 2.0 ** 10, True, values)


@pytest.mark.parametrize("dtype,store,dim", [c for c in CODES if c[0] != F16])
def test_scores_grow_as_scales_fall(A, dtype, store, dim):
    """Every key weighs more than the one before, a little each, and its values are smaller in proportion: the first ones are 2^70 times
    the last ones' and count for no more."""
    lens = [3500]
    cache, pos, crd = make_cache(A, (lens, 1, dim, 16, dtype, store, torch.int32))
    row, place = tokens_of(lens)
    t = place.double()[:, None, None]
    k = (torch.ones(3500, 1, dim, device=DEV) * t * (70 * math.log(2) / 3500) / math.sqrt(dim)).to(dtype)
    v = (normal(2, 3500, 1, dim) * 2.0 ** (20 - 70 * t / 3500)).to(dtype)
    cache.append(k, v, pos, crd, row, place)
    held = [tuple(quantised(x.float(), store).double() for x in (k, v))]
    q = torch.ones(1, 3, dim, device=DEV, dtype=dtype) * torch.tensor([1.0, 0.5, -0.25], device=DEV, dtype=dtype)[:, None]
    held_to(q, A.paged_attention(q, cache, pos, crd, length_of(lens), return_lse=True), held, dim ** -0.5)


@pytest.mark.parametrize("dtype,store,dim", [c for c in CODES if c[0] != F16])
def test_scores_grow_as_scales_fall_in_one_block(A, dtype, store, dim):
    """The same where a block has all keys of a request: 2000 requests that share their pages."""
    n, many = 3500, 2000
    cache, pos, crd = make_cache(A, ([n], 1, dim, 16, dtype, store, torch.int32))
    row, place = tokens_of([n])
    t = place.double()[:, None, None]
    k = (torch.ones(n, 1, dim, device=DEV) * t * (70 * math.log(2) / n) / math.sqrt(dim)).to(dtype)
    v = (normal(2, n, 1, dim) * 2.0 ** (20 - 70 * t / n)).to(dtype)
    cache.append(k, v, pos, crd, row, place)
    held = [tuple(quantised(x.float(), store).double() for x in (k, v))]
    q = torch.ones(1, 3, dim, device=DEV, dtype=dtype) * torch.tensor([1.0, 0.5, -0.25], device=DEV, dtype=dtype)[:, None]
    each = int(pos[1])
    out, lse = A.paged_attention(q.expand(many, -1, -1), cache, torch.arange(many + 1, device=DEV, dtype=torch.int32) * each, crd[:each].repeat(many),
                                 length_of([n] * many), return_lse=True)
    for r in (0, 1, 999, 1998):
        held_to(q, (out[r:r + 1], lse[r:r + 1]), held, dim ** -0.5)


@pytest.mark.parametrize("n,at", [(100, 1), (100, 98), (4000, 1)])
@pytest.mark.parametrize("power", [0, 28, 40, 60])
@pytest.mark.parametrize("dtype,store,dim", [c for c in CODES if c[0] != F16])
def test_equal_weights_beside_a_large_scale(A, dtype, store, dim, power, n, at):
    """All keys are zero but one, of weight e^-80 of the others' and values 2^power times theirs: out is the others' mean, to the bound of
    a sum of equal weights."""
    cache, pos, crd = make_cache(A, ([n], 1, dim, 16, dtype, store, torch.int32))
    row, place = tokens_of([n])
    k, v = torch.zeros(n, 1, dim, device=DEV, dtype=dtype), normal(2, n, 1, dim)
    k[at] = -80 / math.sqrt(dim)
    v[at] *= 2.0 ** power
    v = v.to(dtype)
    cache.append(k, v, pos, crd, row, place)
    held = quantised(v.float(), store).double()
    out, lse = A.paged_attention(torch.ones(1, 3, dim, device=DEV, dtype=dtype), cache, pos, crd, length_of([n]), return_lse=True)
    rest = torch.cat([held[:at], held[at + 1:]])[:, 0]
    want, size, beside = rest.mean(0), rest.abs().mean(0), held[at, 0].abs() * math.exp(-79) / (n - 1)
    bound = ((n + 64) * 4 * E + WEIGHT[dtype]) * size + U[dtype] * want.abs() + beside + TINY[dtype]
    assert bool(((out[0].double() - want).abs() <= bound).all())
    assert bool(((lse[0].double() - math.log(n - 1)).abs() <= (n + 64) * E + 4 * E * math.log(n)).all())
