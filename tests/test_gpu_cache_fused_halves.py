"""Keys normalised, rotated in halves and quantised on their way to the cache: each is off from the formula by half a step of its code, and
by the rounding of what is quantised."""
import pytest
import torch

from tests.test_gpu_attention import CACHE, DEV, E, E4M3, F32, I8, forward64, make_cache, normal, partners, quantised, tables, tokens_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("part", [False, True])
@pytest.mark.parametrize("c", [c for c in CACHE if c[2] % 4 == 0], ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_append_norm_rope_halves(c, part):
    from lapis_b200 import attention as A
    lens, heads, dim, page, dtype, store, idx = c
    rot = dim // 2 if part else dim
    cache, pos, crd = make_cache(A, c)
    row, place = tokens_of(lens, idx)
    x = normal(1, len(row), 5 * heads, dim).to(dtype)
    q, k, v = x[:, :3 * heads], x[:, 3 * heads:4 * heads], x[:, 4 * heads:]
    w = (1 + 0.3 * normal(2, 2, dim)).to(dtype)
    cos, sin = tables(300, rot)
    got_q = cache.append_norm_rope(q, k, v, w[0], w[1], cos, sin, pos, crd, row, place, eps=1e-5)
    want_q, want_k = A.qk_norm_rope(q, k, w[0], w[1], cos, sin, place, eps=1e-5)
    assert torch.equal(got_q, want_q)
    got_k, got_v = cache.read(pos, crd, row, place, dtype=F32)
    assert torch.equal(got_v, quantised(v.float(), store))
    if store not in (I8, E4M3):
        assert torch.equal(got_k, want_k.float())
        return
    exact = forward64(k, w[1], cos, sin, place.long(), 1e-5, False)
    most, off = exact.abs().amax(-1, keepdim=True), (dim + 32) * E * partners(exact, rot, False)
    step = most / 127 * 0.5 if store == I8 else torch.maximum(exact.abs() * 2.0 ** -4, most / 448 * 2.0 ** -10)
    assert bool(((got_k.double() - exact).abs() <= step * (1 + 1e-4) + off + 2 * E * exact.abs()).all())
