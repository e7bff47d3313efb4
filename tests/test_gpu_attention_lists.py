"""Page lists whose pos says more than there is: a request's list ends where the lists do, and one that begins before them is empty."""
import math

import pytest
import torch

from tests.test_gpu_attention import BF16, DEV, E4M3, F16, F32, attend64, fill, holds, make_cache, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("idx,far", [(torch.int32, 2 ** 31 - 1), (torch.int64, 2 ** 62), (torch.int32, 11)])
@pytest.mark.parametrize("dtype,store,dim", [(BF16, BF16, 128), (F16, E4M3, 64), (F32, F32, 20), (F32, F32, 7)])
def test_lists_end_where_there_is_no_more(dtype, store, dim, idx, far):
    from lapis_b200 import attention as A
    lens = [40, 32, 16]
    cache, pos, crd = make_cache(A, (lens, 2, dim, 8, dtype, store, idx), extra=0)
    held = fill(cache, pos, crd, lens, 11, dtype)
    q = normal(5, 3, 4, dim).to(dtype)
    length = torch.full((3,), 2 ** 31 - 1, device=DEV, dtype=idx)
    want = attend64(q, held, dim ** -0.5, 0)
    wrong = pos.clone()
    wrong[3] = far
    holds(q, A.paged_attention(q, cache, wrong, crd, length, return_lse=True), want)
    wrong[0], wrong[1] = -far, -1   # lists that begin before the first entry; the second one of these ends where it did
    out, lse = A.paged_attention(q, cache, wrong, crd, length, return_lse=True)
    assert float(out[:2].abs().max()) == 0 and bool((lse[:2] == -math.inf).all())
    holds(q[2:], (out[2:], lse[2:]), [x[2:] for x in want])
