"""Rows whose largest magnitude is so small that largest code / magnitude does not fit 32 bits are quantised like any other.

Bounds: a code is the rounding of x * (largest / amax), a quotient and a product in 32 bits: off by 2 E of it before its own
rounding (int8: to a half; e4m3: to 2^-4 of it, 2^-10 below its normal numbers).  A scale is a quotient in 32 bits, off by E of
it or, below the normal numbers, by 2^-150."""
import numpy as np
import pytest
import torch

from tests.test_gpu_attention import BF16, DEV, E, E4M3, F32, I8, make_cache, quantised, tables, tokens_of

pytestmark = pytest.mark.gpu

AMPLITUDES = [1.0, 1e-30, 2e-36, 1e-36, 3e-37, 1e-37, 1e-38, 1e-40, 3e-44]


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dim,odd", [(64, False), (64, True), (20, False), (256, False)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [I8, E4M3])
def test_small_rows(store, dtype, dim, odd, fused):
    from lapis_b200 import attention as A
    lens, heads = [len(AMPLITUDES)], 3
    cache, pos, crd = make_cache(A, (lens, heads, dim, 4, dtype, store, torch.int32))
    row, place = tokens_of(lens)
    rng = np.random.default_rng(5)
    x = rng.standard_normal((lens[0], 2 * heads, dim + (1 if odd else 0))) * np.array(AMPLITUDES)[:, None, None]
    x[:, :, 1::3] = 0
    x = torch.from_numpy(x).to(dtype).to(DEV)
    k, v = x[:, :heads, :dim], x[:, heads:, :dim]
    if fused:
        cos, sin = tables(lens[0], dim)
        one = torch.ones(dim, device=DEV)
        cache.append_norm_rope(k, k, v, one, one, cos, sin, pos, crd, row, place, eps=1e-5)
    else:
        cache.append(k, v, pos, crd, row, place)
    page, slot = crd.long()[place.long() // 4], place.long() % 4
    big = 127.0 if store == I8 else 448.0
    for of, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        if fused and of is k:
            continue
        of = of.double().cpu()
        code = (codes.view(torch.uint8)[page, :, slot].view(store)).cpu().float().double()
        scale = scales[page, :, slot].cpu().double()
        most = of.abs().amax(-1)
        want = torch.where(of == 0, 0.0, of * (big / most[..., None]))
        off = torch.full_like(want, 0.5) if store == I8 else torch.clamp(want.abs() * 2.0 ** -4, min=2.0 ** -10)
        assert bool(((code - want).abs() <= off * (1 + 2 * E) + 2 * E * want.abs() + 1e-9).all())
        assert bool(((scale - most / big).abs() <= E * most / big + 2.0 ** -150).all())
        assert bool((code[of == 0] == 0).all())
    got = cache.read(pos, crd, row, place, dtype=F32)[1].cpu().double()
    assert bool(((got - v.double().cpu()).abs() <= off * most[..., None] / big * (1 + 2 * E) + 5 * E * v.double().cpu().abs() + big * 2.0 ** -150 + 2.0 ** -149).all())
    ordinary = quantised(v[:2].float(), store)
    assert torch.equal(cache.read(pos, crd, row[:2], place[:2], dtype=F32)[1], ordinary)
