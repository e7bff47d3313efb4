"""Weights of 4 bits on other streams than the one they were laid out on."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
DEV = "cuda"


def test_weights_outlive_work_on_another_stream():
    """The memory of weights that are dropped while another stream multiplies by them is not given to anyone before that has ended."""
    from lapis_b200 import experts as X
    codes = torch.full((4096, 2048), 0x99, dtype=torch.uint8, device=DEV)
    scale = torch.ones(4096, 32, dtype=BF16, device=DEV)
    x = torch.ones(4, 4096, dtype=BF16, device=DEV)
    busy = torch.ones(8192, 8192, device=DEV)
    out = torch.empty_like(busy)
    side = torch.cuda.Stream()
    X.Int4Matrix(codes, scale, columns=4096).matmul(x), torch.mm(busy, busy, out=out)  # loads the kernels
    matrix = X.Int4Matrix(codes, scale, columns=4096)
    size = matrix._packed.numel()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    with torch.cuda.stream(side):
        for _ in range(8):
            torch.mm(busy, busy, out=out)  # tens of milliseconds
        y = matrix.matmul(x)
    del matrix
    others = [torch.full((size,), 0x55, dtype=torch.uint8, device=DEV) for _ in range(40)]  # the next ones to ask for memory
    torch.cuda.synchronize()
    assert bool((y == 4096).all())
    del others
