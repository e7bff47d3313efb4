"""Smallest values times 4-bit weights: the tensor cores take subnormal numbers of 16 bits as they are, so 16-bit values come out unchanged, and
float32 values in three parts of bf16 lose what lies below the last of its subnormal numbers, 2^-133."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module")
def identity():
    """w = 1 on the diagonal: code 9 less 8, scale 1."""
    from lapis_b200 import experts as X
    codes = torch.full((128, 64), 0x88, dtype=torch.uint8, device=DEV)
    i = torch.arange(128, device=DEV)
    codes[i, i // 2] = torch.where(i % 2 == 0, 0x89, 0x98).to(torch.uint8)
    return X.Int4Matrix(codes, torch.ones(128, 2, device=DEV), columns=128, group=64)


@pytest.mark.parametrize("rows", [1, 2, 8, 9, 40])
@pytest.mark.parametrize("dtype,bits", [(torch.float16, 10), (torch.bfloat16, 7)], ids=str)
def test_subnormal_values_of_16_bits(identity, dtype, bits, rows):
    x = torch.from_numpy(np.random.default_rng(rows).integers(1, 2 ** bits, (rows, 128)).astype(np.int16)).to(DEV).view(dtype)
    assert torch.equal(identity.matmul(x), x) and torch.equal(identity.matmul(-x), -x)


@pytest.mark.parametrize("rows", [1, 2, 3, 40])
@pytest.mark.parametrize("exponent", [-149, -140, -133, -127, -126, -120, -111, -110, -109, -103])
def test_small_values_of_32_bits(identity, exponent, rows):
    """From 2^-110 on all 24 bits are at 2^-133 or above."""
    x = torch.from_numpy(np.ldexp(np.random.default_rng(rows).uniform(1, 2, (rows, 128)), exponent).astype(np.float32)).to(DEV)
    off = (identity.matmul(x).double() - x.double()).abs().max()
    assert float(off) < 2.0 ** -133 if exponent < -110 else float(off) == 0.0
