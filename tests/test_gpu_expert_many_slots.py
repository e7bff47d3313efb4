"""Lists of very many slots: right, and in time that grows as they do."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("tokens,k,experts", [(4_200_001, 1, 1024), (1_000_003, 9, 3), (5_000_011, 8, 300)])
def test_lists_of_millions(tokens, k, experts):
    """From about five million slots on a block takes several rounds."""
    from lapis_b200 import experts as X
    gen = torch.Generator(DEV).manual_seed(k)
    expert = torch.randint(-1, experts + 1, (tokens, k), generator=gen, device=DEV, dtype=torch.int32)
    lists = X.ExpertLists(expert, experts)
    bucket = torch.where((expert >= 0) & (expert < experts), expert, experts).flatten()
    order = torch.sort(bucket, stable=True).indices
    count = torch.bincount(bucket, minlength=experts + 1).cumsum(0)
    assert lists.pos[0] == 0 and torch.equal(lists.pos[1:].long(), count[:experts])
    assert torch.equal(lists.crd.long(), order)
    assert torch.equal(lists.place.flatten().long()[order], torch.arange(tokens * k, device=DEV))


def test_time_grows_with_the_slots():
    """2^26 slots are 16 times 2^22.  With every block reading the counts of a block for each 16,384 slots they took 84 times as long."""
    from lapis_b200 import experts as X
    took = []
    for slots in (2 ** 22, 2 ** 26):
        expert = torch.randint(0, 256, (slots // 8, 8), generator=torch.Generator(DEV).manual_seed(1), device=DEV, dtype=torch.int32)
        X.ExpertLists(expert, 256)
        times = []
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            begin.record()
            X.ExpertLists(expert, 256)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        took.append(min(times))
    assert took[1] <= 40 * took[0]
