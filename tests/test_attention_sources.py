"""The kernels around attention become resident while the launch in front of them still writes (launch_pdl): none of their operands
may come by the read-only path, and each of them waits before it touches memory.  A stale read cannot be provoked, so the
sources are looked at."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lapis_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


@pytest.mark.parametrize("name", ["attention.cu", "rotate.cu", "kv.h"])
def test_no_read_only_loads(name):
    text = _source(name)
    assert "__ldg" not in text and "__restrict__" not in text and "ld.global.nc" not in text


@pytest.mark.parametrize("name", ["attention.cu", "rotate.cu"])
def test_kernels_that_overlap_wait(name):
    text = _source(name)
    for kernel in set(re.findall(r"launch_pdl\((\w+)", text)):
        bodies = re.findall(r"__global__ void __launch_bounds__\([^\n]*?\)\s+%s\(.*?\n}\n" % kernel, text, flags=re.S)
        assert len(bodies) == 1, kernel
        assert bodies[0].count("pdl_wait();") == 1, kernel
