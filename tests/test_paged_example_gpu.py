"""The example: page_step, rotary_append and paged_attention together, as a CUDA graph, against the same without a cache."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompts,steps", [((5, 33, 1, 70), 8), ((16,), 33), ((1, 2, 3, 15, 16, 17, 31, 32), 5)])
def test_paged_decoding(prompts, steps):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decoding.py")
    spec = importlib.util.spec_from_file_location("paged_decoding", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main(steps, prompts, check=True)
    assert got["lengths"] == [p + steps for p in prompts]
    assert got["pages"] == sum(-(-(p + steps) // example.PAGE) for p in prompts)
    # (a step's bf16 outputs and those without a cache are rounded apart at every product of two layers: a few roundings of 2^-8 of the largest)
    assert got["worst"] <= 6 * 2.0 ** -8
