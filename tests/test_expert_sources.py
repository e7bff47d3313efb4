"""The kernels of a layer of experts become resident while the launch in front of them still writes (launch_pdl): none of their operands
may come by the read-only path, and each of them waits before it touches memory that a launch in front may write.  A stale read cannot be
provoked, nor can two clusters that wait for each other's tensor memory, so the sources are looked at."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lapis_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


@pytest.mark.parametrize("name", ["experts.cu", "experts.h", "int4.cu", "int4.h", "int4_few.cu", "int4_many.cu"])
def test_no_read_only_loads(name):
    text = _source(name)
    assert "__ldg" not in text and "__restrict__" not in text and "ld.global.nc" not in text


@pytest.mark.parametrize("name,kernels", [
    ("experts.cu", {"route_kernel", "route_backward_kernel", "list_count_kernel", "list_place_kernel", "gather_kernel", "combine_ring_kernel", "combine_kernel",
                    "combine_backward_kernel", "gather_narrow_kernel", "combine_narrow_kernel", "combine_backward_narrow_kernel"}),
    ("int4_few.cu", {"int4_few_kernel"}),
    ("int4_many.cu", {"arrange_kernel", "int4_many_kernel"}),
])
def test_kernels_that_overlap_wait(name, kernels):
    bodies = dict(re.findall(r"__global__ void __launch_bounds__\([^\n]*?\)\s+(\w+)\((.*?\n}\n)", _source(name), flags=re.S))
    assert set(bodies) == kernels
    for body in bodies.values():
        assert body.count("pdl_wait();") == 1


def test_tensor_memory_is_asked_for_in_turn():
    """Behind pdl_wait(), so that no CTA holds it that waits for the launch in front, and in front of pdl_release(), so that the launch behind
    takes none that this one still needs."""
    text = _source("int4_many.cu")
    body = text[text.index("int4_many_kernel(const"):]
    alloc = body.index("tcgen05.alloc")
    assert body.index("pdl_wait();") < alloc < body.rindex("pdl_release();")
    # two CTAs of 256 columns or one of 512 fit an SM's shared memory (228 KB, one of them kept back for each), and nothing beside them
    sizes = [int(n) for n in re.search(r"== 256 \? (\d+) << 10 : (\d+) << 10", text).groups()]
    room = 228
    assert 2 * (sizes[0] + 1) <= room < 3 * (sizes[0] + 1) and sizes[1] + 1 <= room < sizes[0] + sizes[1] + 2
