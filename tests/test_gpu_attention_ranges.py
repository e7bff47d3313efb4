"""Attention over quantised and 16-bit caches where scores, values and scales lie far apart: against 64 bits, with the bounds of
test_gpu_attention.py where none is derived here."""
import math

import pytest
import torch

from tests.test_gpu_attention import BF16, DEV, E4M3, F16, F32, I8, U, WEIGHT, attend64, holds, make_cache, normal, quantised, tokens_of

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
