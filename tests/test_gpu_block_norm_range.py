"""The norms around a block where a row's squares leave fp32's range although their mean does not.

Rows hold one magnitude, or one value beside zeros, so the exact results are short; the bound of every other row applies:
a row's factor is off by ROW (test_gpu_block_norm), a rounding to bf16 by 2^-8 of the value."""
import pytest
import torch

import block_helpers as H
from test_gpu_block_norm import ROW, _reference

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def qf():
    import qwen_fastpath
    return qwen_fastpath


def _signs(M, N):
    return torch.where(torch.rand(M, N, generator=H.gen(N)) < 0.5, -1.0, 1.0)


@pytest.mark.parametrize("N", [8, 64, 256, 520, 5120, 8200, 16392, 32768])
@pytest.mark.parametrize("wide", [False, True])
def test_even_rows(qf, N, wide):
    """Squares of 2^126.6 and a mean as large: two of them no longer add up to a number."""
    x = (1.1e19 * _signs(3, N)).to(BF16)
    r = torch.zeros(3, N, dtype=F32 if wide else BF16)
    w = torch.ones(N, dtype=BF16)
    y, h = qf.block_norm_rows(x.cuda(), r.cuda(), w.cuda(), w.cuda(), alpha=0.75)
    ry, rh, by, bh = _reference(x, r, w, w, None, "none", 0.75, 1e-6, 0.0)
    H.within(y, ry, by, H.F32 if wide else H.BF16)
    H.within(h, rh, bh, H.BF16)


@pytest.mark.parametrize("N,top", [(64, 66), (520, 68), (5120, 70), (8200, 70), (16392, 70), (32768, 71)])
def test_one_value_beside_zeros(qf, N, top):
    """A single square past 2^128, its mean below."""
    assert 2 * top >= 128 and 2.0 ** (2 * top) / N < 2.0 ** 128
    x = torch.zeros(2, N, dtype=BF16)
    x[0, 3] = 2.0 ** top
    x[1, N - 1] = -(2.0 ** top)
    r, w = torch.zeros(2, N), torch.ones(N, dtype=BF16)
    y, h = qf.block_norm_rows(x.cuda(), r.cuda(), w.cuda(), None)
    ry, rh, by, bh = _reference(x, r, w, None, None, "none", 1.0, 1e-6, 0.0)
    H.within(y, ry, by, H.F32)
    H.within(h, rh, bh, H.BF16)


@pytest.mark.parametrize("N", [8, 256, 5120, 8200, 32768])
def test_second_norm(qf, N):
    """The same for the sum: an fp32 residual of 2^63.25."""
    x = torch.zeros(2, N, dtype=BF16)
    r = 1.1e19 * _signs(2, N)
    y, h = qf.block_norm_rows(x.cuda(), r.cuda())
    assert torch.equal(y.cpu(), r)
    ry, rh, by, bh = _reference(x, r, None, None, None, "none", 1.0, 1e-6, 0.0)
    H.within(h, rh, bh, H.BF16)


def test_not_finite_rows_stay_as_they_were(qf):
    x = torch.ones(4, 520, dtype=BF16)
    x[0, 9] = float("inf")
    x[1, 9] = float("nan")
    x[2] = 3e38  # a mean past fp32: its reciprocal root is zero
    r, w = torch.ones(4, 520), torch.ones(520, dtype=BF16)
    y, h = (t.cpu().float() for t in qf.block_norm_rows(x.cuda(), r.cuda(), w.cuda()))
    others = torch.arange(520) != 9
    assert torch.isnan(y[0, 9]) and y[0, others].eq(1).all() and torch.isnan(h[0]).all()
    assert torch.isnan(y[1]).all() and torch.isnan(h[1]).all()
    assert y[2].eq(1).all()
    assert ((y[3] - 2).abs() <= 2 * ROW + 2 * 1e-6 + 2.0 ** -22).all()


@pytest.mark.parametrize("N", [64, 136, 256, 520])
def test_neighbours_keep_their_bits(qf, N):
    """Rows that share a wavefront with one whose squares are taken again, tiny ones among them."""
    g = H.gen(N)
    x = H.rows(g, 16, N)
    x[3] *= 2.0 ** -60
    r, w = torch.randn(16, N, generator=g), torch.ones(N, dtype=BF16)
    want = qf.block_norm_rows(x.cuda(), r.cuda(), w.cuda(), w.cuda(), eps=0.0)
    x[5] = 1.1e19
    got = qf.block_norm_rows(x.cuda(), r.cuda(), w.cuda(), w.cuda(), eps=0.0)
    others = torch.arange(16) != 5
    for a, b in zip(want, got):
        assert torch.equal(a.cpu()[others], b.cpu()[others]) and torch.isfinite(b).all()
