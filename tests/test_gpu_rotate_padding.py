"""Norms with rotation and an eps of zero: what is no row (padding, and the lanes beside the last head) adds nothing to the gradients.

Bounds as in test_gpu_attention.py, with eps = 0 in the formulas; a double eps below 2^-150 is zero in 32 bits."""
import pytest
import torch

from tests.test_gpu_attention import BF16, E, F16, F32, TINY, U, backward64, forward64, normal, partners, rotate_inputs

pytestmark = pytest.mark.gpu

CASES = [
    # tokens, q heads, k heads, dim, rot, pairs, type, weights, indices
    (9, 5, 3, 128, 128, "half", BF16, BF16, torch.int32),
    (6, 1, 2, 128, 64, "near", BF16, F32, torch.int64),
    (7, 3, 1, 256, 256, "half", F16, F16, torch.int32),
    (6, 1, 5, 64, 64, "near", F32, F32, torch.int32),
    (2000, 3, 1, 32, 32, "half", BF16, BF16, torch.int32),
]


@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("strided", ["no", "view", "odd"])
@pytest.mark.parametrize("c", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_rotate_without_eps(c, strided, eps):
    from lapis_b200 import attention as A
    q, k, qw, kw, cos, sin, place, near = rotate_inputs(c, strided)
    place[1], place[4] = -1, 50
    real = (place >= 0) & (place < 50)
    at = place[real].long()
    dq, dk = normal(5, *q.shape).to(q.dtype), normal(6, *k.shape).to(q.dtype)
    got = A.qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, place, eps=eps, interleaved=near)
    out = A.qk_norm_rope(q, k, qw, kw, cos, sin, place, eps=eps, interleaved=near)
    dim = q.shape[2]
    for x, w, dy, dx, dw, y in ((q, qw, dq, got[0], got[2], out[0]), (k, kw, dk, got[1], got[3], out[1])):
        assert float(dx[~real].abs().max()) == 0 and float(y[~real].abs().max()) == 0
        x, dy, dx, y = x[real], dy[real], dx[real], y[real]
        want = forward64(x, w, cos, sin, at, 0.0, near)
        n = x.double() / x.double().square().mean(-1, keepdim=True).sqrt() * w.double()
        assert bool(((y.double() - want).abs() <= U[x.dtype] * want.abs() + TINY[x.dtype] + (dim + 16) * E * partners(n, c[4], near)).all())
        want, want_w, dn, r = backward64(dy, x, w, cos, sin, at, 0.0, near)
        g = partners(dy.double(), c[4], near) * w.double().abs()
        size = r * (g + x.double().abs() * r * r * (g * x.double().abs()).mean(-1, keepdim=True))
        assert bool(((dx.double() - want).abs() <= U[x.dtype] * want.abs() + TINY[x.dtype] + (2 * dim + 32) * E * size).all())
        terms = (partners(dy.double(), c[4], near) * x.double().abs() * r).sum((0, 1))
        assert bool(((dw.double() - want_w).abs() <= (x.shape[0] * x.shape[1] + dim + 32) * E * terms).all())
