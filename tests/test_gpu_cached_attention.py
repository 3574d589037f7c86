"""examples/cached_attention.py: projections, norms and rotation, cache and attention as one path."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("bits", [4, 8])
def test_example_agrees_with_dense_attention(bits):
    """Relative to the largest output of a head, bf16 rounding of the result is 2^-9 to 2^-8; the weights' fp16
    rounding adds 2^-11 of the weighted values."""
    spec = importlib.util.spec_from_file_location("cached_attention", os.path.join(ROOT, "examples", "cached_attention.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert 0.0 < mod.main(bits) <= 2.0 ** -8 + 2.0 ** -9
