"""Arguments that do not fit the C descriptors are refused as the others are."""
import pytest

pytestmark = pytest.mark.gpu

import torch
import annc_b200  # noqa: F401,E402  (no fallback: a missing library fails the collection)
from annc_b200 import AnncError, device  # noqa: E402


@pytest.mark.parametrize("scale", [1e39, -1e39, float("inf"), float("-inf"), float("nan")])
def test_scales_that_are_no_finite_f32(scale):
    q, k = torch.zeros((2, 4, 64), device="cuda", dtype=torch.bfloat16), torch.zeros((9, 2, 64), device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 3.0)
    with pytest.raises(AnncError):
        device.PrefixAttention(4, 2, 64, 2).run(q, k, k, out, scale=scale)
    assert bool((out == 3).all())
