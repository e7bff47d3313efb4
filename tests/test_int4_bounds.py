"""The bound of tests/int4_sums.py, on the CPU: a product computed as the kernels compute it stays within, one that loses a part of x, a column
or the precision of its sums does not."""
import numpy as np
import pytest
import torch

from tests import int4_sums


def cut(a, last):
    """Towards zero to multiples of `last`."""
    return np.trunc(a / last) * last


def cut_sum(addends):
    """Their sum (axis 0) as a tensor core forms it: each cut at 2^-23 of the largest one's power of two, the sum cut to 24 bits."""
    most = np.abs(addends).max(0)
    last = np.where(most > 0, np.exp2(np.floor(np.log2(np.where(most > 0, most, 1.0))) - 23), 1.0)
    total = cut(addends, last).sum(0)
    size = np.where(total != 0, np.abs(total), 1.0)
    return cut(total, np.exp2(np.floor(np.log2(size)) - 23))


def parts_of(x, parts):
    """bf16 parts of 32-bit values, cut; other types are one."""
    if x.dtype != torch.float32:
        return [x.double().numpy()]
    got, left = [], x.numpy().copy()
    for _ in range(parts):
        p = (left.view(np.uint32) & 0xffff0000).view(np.float32)
        got.append(p.astype(np.float64))
        left = left - p
    return got


def kernel(x, number, scale, group, parts=3, lost=None, sums=np.float32):
    """x [rows, columns] times number [outputs, columns] * scale [outputs, groups]."""
    rows, columns = x.shape
    y = np.zeros((rows, number.shape[0]), np.float32)
    for p in reversed(parts_of(x, parts)):  # the small parts first
        if lost is not None:
            p = p.copy()
            p[:, lost] = 0
        of_part = np.zeros_like(y)
        for g in range(scale.shape[1]):
            acc = np.zeros((rows, number.shape[0]))
            for c in range(g * group, min((g + 1) * group, columns), 16):
                n = slice(c, min(c + 16, (g + 1) * group, columns))
                acc = cut_sum(np.concatenate([acc[None], np.einsum("rc,oc->cro", p[:, n], number[:, n])]))
            acc = acc.astype(np.float32).astype(sums).astype(np.float64)
            of_part = (of_part + scale[:, g].astype(np.float64) * acc).astype(np.float32)
        y = y + of_part
    return torch.from_numpy(y).to(x.dtype)


@pytest.mark.parametrize("dtype", list(int4_sums.U), ids=str)
@pytest.mark.parametrize("shape", [s for s in int4_sums.SHAPES if s[2] != 9000 or s[0] == 1], ids=str)
def test_bound(shape, dtype):
    rows, outputs, columns, group, zeros = shape
    rows, outputs = min(rows, 6), min(outputs, 60)  # an element's error does not depend on the others
    rng = np.random.default_rng(columns)
    number = rng.integers(0, 16, (outputs, columns)) - 8.0
    scale = torch.from_numpy(rng.uniform(-0.1, 0.3, (outputs, -(-columns // group)))).to(dtype)
    x = torch.from_numpy(rng.standard_normal((rows, columns)) * columns ** -0.5).to(dtype)
    w = torch.from_numpy(number * scale.double().numpy().repeat(group, 1)[:, :columns])
    scale = scale.float().numpy()

    assert int4_sums.near(kernel(x, number, scale, group), x, w, group)
    assert not int4_sums.near(kernel(x, number, scale, group, lost=columns // 2), x, w, group)
    if dtype == torch.float32:
        assert not int4_sums.near(kernel(x, number, scale, group, parts=2), x, w, group)
        assert not int4_sums.near(kernel(x, number, scale, group, sums=np.float16), x, w, group)
