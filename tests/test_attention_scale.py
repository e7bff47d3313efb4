"""Scales that are numbers of 64 bits but, times log2 e, not of 32: refused, without a GPU."""
import ctypes

import pytest

from lapis_b200 import _lib
from tests.test_attention_arguments import BADARG, BF16, CACHE, HEADS, LISTS, ref


@pytest.mark.parametrize("scale", [1e39, -1e39, 3e38, 1.7e308])
def test_scales_beyond_32_bits_are_refused(scale):
    lib = _lib.load()
    assert lib.lapis_b200_paged_attention(BF16, 3, ref(HEADS), ref(CACHE), ref(LISTS), 64, ctypes.c_double(scale), 0, 64, None, None) == BADARG
    assert b"scale" in lib.lapis_last_error_message()
