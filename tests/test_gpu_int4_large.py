"""Products with 4-bit weights whose operands or results are larger than 32-bit offsets reach."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
DEV = "cuda"


@pytest.mark.parametrize("tokens", [160, 6000])
def test_weights_of_gigabytes(tokens):
    """160 experts of 8192 x 8192, 5.4 GB of codes; few rows of each expert, and many."""
    from lapis_b200 import experts as X
    experts, outputs, columns = 160, 8192, 8192
    gen = torch.Generator(DEV).manual_seed(1)
    codes = torch.randint(0, 256, (experts, outputs, columns // 2), generator=gen, device=DEV, dtype=torch.uint8)
    scale = torch.rand(experts, outputs, columns // 128, generator=gen, device=DEV).to(BF16)
    matrix = X.Int4Matrix(codes, scale, columns=columns)
    lists = X.ExpertLists((torch.arange(tokens, device=DEV) % experts)[:, None], experts)
    x = torch.randn(tokens, columns, generator=gen, device=DEV).to(BF16)
    y, pos = matrix.matmul(x, lists, fetch=True), lists.pos.tolist()
    for e in (0, 63, 64, 127, 128, 159):
        alone = X.Int4Matrix(codes[e].clone(), scale[e].clone(), columns=columns)
        rows = x[lists.crd[pos[e]:pos[e + 1]].long()]
        want = alone.matmul(rows)
        # the same sums, but for how many shares a tile has: 32 bits, rounded to the same or the next of 8 bits
        assert float((y[pos[e]:pos[e + 1]].float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
        assert float((y[pos[e]:pos[e + 1]] != want).float().mean()) < 0.01


def test_results_of_gigabytes():
    """140,000 rows of 16,384 values."""
    from lapis_b200 import experts as X
    gen = torch.Generator(DEV).manual_seed(2)
    codes = torch.randint(0, 256, (16384, 32), generator=gen, device=DEV, dtype=torch.uint8)
    matrix = X.Int4Matrix(codes, torch.ones(16384, 1, device=DEV, dtype=BF16), columns=64)
    x = torch.randint(-3, 4, (140_000, 64), generator=gen, device=DEV).to(BF16)  # whole numbers: exact in any order
    y = matrix.matmul(x)
    for at in (0, 70_000, 131_070, 139_990):
        assert torch.equal(y[at:at + 10], matrix.matmul(x[at:at + 10].clone()))
