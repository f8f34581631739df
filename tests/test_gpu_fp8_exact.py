"""Block-scaled FP8 products with integers, bit for bit, in every form of the kernels (exact_cases)."""
import pytest
import torch

import exact_cases as X

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def qf():
    import qwen_fastpath
    return qwen_fastpath


def _check(qf, layout, M, N, K, a8):
    x, q, s, bias, xd = X.product(M, N, K, a8)
    x, q, s, bias = (t.cuda() for t in (x, q, s, bias))
    want = X.reference(xd.cuda(), q, s, bias)
    w = qf.fp8_to_tiled(q.t()) if layout else q.t()
    mm = qf.fp8_w8a8_mm if a8 else qf.fp8_w8a16_mm
    for out in (F32, BF16):
        y = mm(x, w, s, out, bias, N)
        wrong = (y != want.to(out)).nonzero()
        assert not len(wrong), f"{len(wrong)} of {y.numel()} {out} values differ, the first at {wrong[0].tolist()}"


@pytest.mark.parametrize("layout,M,N,K", X.DECODE)
def test_decode(qf, layout, M, N, K):
    _check(qf, layout, M, N, K, False)


@pytest.mark.parametrize("layout,M,N,K", X.W8A8)
def test_w8a8(qf, layout, M, N, K):
    _check(qf, layout, M, N, K, True)
