"""Outputs of one head a token that reach over more than 2^31 values."""
import pytest
import torch

import kv4_helpers as H
import qwen_fastpath as qf
from test_gpu_kv4_attention import _batch, _call

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
APART = 2 ** 30 + 64  # values from token to token


@pytest.fixture(scope="module")
def room():
    return torch.empty(2 * APART + 256, dtype=BF16, device="cuda")


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention(room, D):
    s = _batch(D, [50], [3], 1, 1, D, 16)
    out = room.as_strided((3, 1, D), (APART, D, 1))
    assert _call(s, out=out) is out
    assert torch.equal(out, _call(s))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_norms_and_rotation(room, D):
    g = H.gen(D)
    x, y = (torch.randn(3, 1, D, generator=g).to(BF16).cuda() for _ in range(2))
    weight = torch.randn(D, generator=g).to(BF16).cuda()
    out = room.as_strided((3, 1, D), (APART, D, 1))
    want = qf.qk_norm_rope(x, y, None, None, weight, weight)
    got, _ = qf.qk_norm_rope(x, y, None, None, weight, weight, query_out=out)
    assert got is out and torch.equal(out, want[0])
    _, got = qf.qk_norm_rope(x, y, None, None, weight, weight, key_out=out)
    assert got is out and torch.equal(out, want[1])
