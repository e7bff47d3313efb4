"""The operators together, as examples/attention_serving.py runs them."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("requests,prompt", [(1, 5), (7, 300)])
def test_serving_example(cache, requests, prompt):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "attention_serving.py")
    spec = importlib.util.spec_from_file_location("attention_serving", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    us, error, bound = example.serve(requests=requests, prompt=prompt, steps=5, q_heads=8, kv_heads=2, dim=64, width=128, page_size=16, cache_type=cache)
    assert us > 0 and error <= bound
