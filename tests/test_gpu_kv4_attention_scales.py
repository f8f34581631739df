"""Attention over the 4-bit cache with the smallest scales, of queries and keys whose products are near fp32's largest."""
import pytest
import torch

from test_gpu_kv4_attention import BF16, _batch, _call, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.0, -0.0, 2.0 ** -149, -2.0 ** -140, 2.0 ** -126, 2.0 ** -122])
@pytest.mark.parametrize("D,q", [(64, 3), (128, 2), (128, 90), (256, 70)])
def test_scales_of_nearly_nothing(D, q, scale):
    """Scores of about 2^124 before the scale: with one of 0 every position weighs the same, as with one that leaves them below
    2^-10; with 2^-122 they do not."""
    s = _batch(D, [333], [q], 4, 1, D, 16, spread=2.0 ** 61)
    s["query"] = (s["query"].float() * 2.0 ** 58).to(BF16)
    s["scale"] = scale
    _check(s, _call(s))
