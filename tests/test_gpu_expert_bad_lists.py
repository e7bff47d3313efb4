"""Lists that are no lists, on the kernels for many rows of an expert: nothing is followed out of the arrays."""
import ctypes

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype", list(TYPES), ids=str)
def test_bad_lists_of_many_rows(dtype, group):
    from lapis_b200 import experts as X
    from lapis_b200 import _lib
    tokens, k, experts, outputs, columns, ends = 60, 2, 4, 40, 320, 4096
    rng = np.random.default_rng(group)
    codes = torch.from_numpy(rng.integers(0, 256, (experts, outputs, columns // 2), dtype=np.uint8)).to(DEV)
    matrix = X.Int4Matrix(codes, torch.ones(experts, outputs, -(-columns // group), device=DEV), columns=columns, group=group)
    slots = tokens * k
    crds = [torch.arange(slots, dtype=torch.int32), torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31 - 1, slots)).int()]
    poses = [[0, 30, 60, 90, 120], [-7, 2 ** 31 - 1, -2 ** 31, 5, 2 ** 31 - 1], [200, 300, 400, 500, 600], [120, 60, 30, 1, -4], [0, 120, 0, 120, 0]]
    for crd in crds:
        for pos in poses:
            for fetch in (0, 1):
                x = torch.from_numpy(rng.standard_normal((tokens if fetch else slots, columns))).to(DEV, dtype)
                guarded = torch.full((2 * ends + slots * outputs,), 77.0, dtype=dtype, device=DEV)
                arrays = [t.to(DEV) for t in (torch.tensor(pos, dtype=torch.int32), crd, torch.arange(slots, dtype=torch.int32))]
                lists = _lib.ExpertLists(tokens, k, experts, *(t.data_ptr() for t in arrays))
                y = guarded[ends:]
                _lib.check(_lib.load().lapis_b200_int4_matmul(TYPES[dtype], ctypes.byref(matrix._c), x.shape[0], x.data_ptr(), x.stride(0), ctypes.byref(lists), fetch,
                                                              y.data_ptr(), torch.cuda.current_stream().cuda_stream))
                torch.cuda.synchronize()
                assert bool((guarded[:ends] == 77).all()) and bool((guarded[ends + slots * outputs:] == 77).all())
                if pos == poses[0]:
                    row = (arrays[1].long() // k if fetch else torch.arange(slots, device=DEV))
                    there = (row >= 0) & (row < x.shape[0])
                    got = y[:slots * outputs].view(slots, outputs)
                    assert not got[~there].any() and bool(got[there].any(-1).all())
