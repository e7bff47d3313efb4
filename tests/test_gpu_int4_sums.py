"""Sums of products with 4-bit weights: held in 32 bits over thousands of columns (tests/int4_sums.py has the bound and where it comes from),
and exact where every sum is a whole number of 24 bits, whatever the order in which warps, stages and shares of a tile add it."""
import numpy as np
import pytest
import torch

from tests import int4_sums

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEV = "cuda"


@pytest.fixture(scope="module")
def X():
    from lapis_b200 import experts
    return experts


def weights4(seed, experts, outputs, columns, group, zeros, scales):
    """(codes, scales, zeros) and the numbers that they stand for."""
    rng = np.random.default_rng(seed)
    lead = (outputs,) if experts is None else (experts, outputs)
    groups = -(-columns // group)
    codes = torch.from_numpy(rng.integers(0, 256, (*lead, (columns + 1) // 2), dtype=np.uint8)).to(DEV)
    scale = scales(rng, (*lead, groups))
    zero = torch.from_numpy(rng.integers(0, 16, (*lead, groups), dtype=np.uint8)).to(DEV) if zeros else None
    c = torch.arange(columns, device=DEV)
    number = ((codes[..., c // 2].int() >> (4 * (c % 2)).int()) & 15) - (8 if zero is None else zero[..., c // group].int())
    return (codes, scale, zero), number.double() * scale.double()[..., c // group]


def any_scales(dtype):
    return lambda rng, shape: torch.from_numpy(rng.uniform(-0.1, 0.3, shape)).to(DEV, dtype)


def powers_of_two(rng, shape):
    return torch.from_numpy(np.exp2(rng.integers(-3, 1, shape))).to(DEV, F32)


def ones(rng, shape):
    return torch.ones(shape, device=DEV)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("rows,outputs,columns,group,zeros", int4_sums.SHAPES)
def test_sums_are_held_in_32_bits(X, rows, outputs, columns, group, zeros, dtype):
    given, w = weights4(columns, None, outputs, columns, group, zeros, any_scales(dtype))
    x = torch.from_numpy(np.random.default_rng(rows).standard_normal((rows, columns)) * columns ** -0.5).to(DEV, dtype)
    assert int4_sums.near(X.Int4Matrix(*given, columns=columns, group=group).matmul(x), x, w, group)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("rows,outputs,columns,group,zeros", int4_sums.SHAPES)
def test_whole_numbers_are_exact(X, rows, outputs, columns, group, zeros, dtype):
    """Eighths below 9000 x 3 x 15 = 405,000: 22 bits at most, so 32 bits hold every sum and the one rounding is of the exact result."""
    given, w = weights4(rows, None, outputs, columns, group, zeros, powers_of_two)
    x = torch.from_numpy(np.random.default_rng(outputs).integers(-3, 4, (rows, columns))).to(DEV, dtype)
    assert torch.equal(X.Int4Matrix(*given, columns=columns, group=group).matmul(x), (x.double() @ w.T).to(dtype))


@pytest.mark.parametrize("rows,outputs,columns,group,zeros", int4_sums.SHAPES)
def test_numbers_of_18_bits_are_exact(X, rows, outputs, columns, group, zeros):
    """Two values of 18 bits a row, three parts of bf16 each: sums below 2 x 2^18 x 15 < 2^23."""
    given, w = weights4(rows, None, outputs, columns, group, zeros, ones)
    rng = np.random.default_rng(outputs)
    x = torch.zeros(rows, columns, device=DEV)
    for _ in range(2):
        x[torch.arange(rows), torch.from_numpy(rng.integers(0, columns, rows))] = torch.from_numpy(rng.integers(2 ** 17, 2 ** 18, rows) | 1).to(DEV, F32)
    assert torch.equal(X.Int4Matrix(*given, columns=columns, group=group).matmul(x), (x.double() @ w.T).float())


LISTED = [
    # tokens, k, experts, outputs, columns, group, zeros
    (7, 3, 5, 50, 2500, 64, True), (40, 4, 3, 64, 1320, 128, False), (90, 3, 2, 20, 4200, 32, True), (64, 8, 128, 48, 1024, 32, False), (300, 2, 4, 130, 640, 64, False),
]


@pytest.mark.parametrize("fetch", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("tokens,k,experts,outputs,columns,group,zeros", LISTED)
@pytest.mark.parametrize("popular", [False, True])
def test_sums_of_lists(X, popular, tokens, k, experts, outputs, columns, group, zeros, dtype, fetch):
    """Every expert alike, and one that has half of all slots, many times the mean that the kernels are chosen for."""
    rng = np.random.default_rng(tokens)
    expert = rng.integers(-1, experts + 1, (tokens, k))
    if popular:
        expert[rng.random((tokens, k)) < 0.5] = experts - 1
    lists = X.ExpertLists(torch.from_numpy(expert).to(DEV), experts)
    pos = lists.pos.tolist()
    x = torch.from_numpy(rng.standard_normal((tokens if fetch else tokens * k, columns)) * columns ** -0.5).to(DEV, dtype)
    whole = torch.from_numpy(rng.integers(-3, 4, x.shape)).to(DEV, dtype)
    for x, scales in ((x, any_scales(dtype)), (whole, powers_of_two)):
        given, w = weights4(tokens, experts, outputs, columns, group, zeros, scales)
        y = X.Int4Matrix(*given, columns=columns, group=group).matmul(x, lists, fetch=fetch)
        rows = x[lists.crd.long() // k] if fetch else x
        assert not y[pos[-1]:].any()
        for e in range(experts):
            s = slice(pos[e], pos[e + 1])
            if scales is powers_of_two:
                assert torch.equal(y[s], (rows[s].double() @ w[e].T).to(dtype))
            elif pos[e] < pos[e + 1]:
                rms, most = int4_sums.far(y[s], rows[s], w[e], group)
                assert rms <= 1.5 and most <= 6  # from 20 elements on, whose root mean square is off by a sixth
