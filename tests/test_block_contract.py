"""What the W8A8 product says of its own arithmetic, and that it is so: within 8 neighbouring k what lies below
2^(e - 13) is dropped, e the largest sum of two exponents among them; everything else is added whole."""
import os
import re

import pytest
import torch

import block_helpers as H

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "qf_block.h")
BF16, F32 = torch.bfloat16, torch.float32


def test_the_contract_states_it():
    import qwen_fastpath as qf
    text = open(HEADER).read()
    said = " ".join(text[:text.index("int qf_fp8_w8a8_linear(")].rsplit("/*", 1)[1].replace("\n *", " ").split())
    for doc in (said, " ".join(qf.fp8_w8a8_mm.__doc__.split())):
        assert "products are not exact" in doc and "2^(e - 13)" in doc and "1.5e-5 to 3.6e-5" in doc
        assert not re.search(r"(?<!not )exact products|the rest as qf_fp8_w8a16_gemm", doc)
    assert "exact products" in qf.fp8_w8a16_mm.__doc__


def _one_block(xs, ws):
    """x bf16 [32, 128] and w e4m3 [32, 128], the rows alike: 448 at k = 127 keeps x's scale at 1 (w is 0 there)."""
    x, w = torch.zeros(32, 128), torch.zeros(32, 128)
    x[:, :len(xs)], w[:, :len(ws)] = torch.tensor(xs), torch.tensor(ws)
    x[:, 127] = 448.0
    return x.to(BF16).cuda(), w.to(H.FP8).cuda(), torch.ones(1, 1, device="cuda")


# a group of 8: (x, w), its exact sum, and what may be dropped (7 products below 2^(e - 13))
@pytest.mark.gpu
@pytest.mark.parametrize("xs,ws,loss", [
    ([448.] + [8.] * 7, [448.] + [1.] * 7, 0.0),              # e = 16: multiples of 8 are kept
    ([448.] + [4.] * 7, [448.] + [1.] * 7, 7 * 8.0),
    ([448.] + [1.] * 7, [448.] + [0.875] * 7, 7 * 8.0),
    ([448., -448.] + [3.] * 6, [448., 448.] + [1.5] * 6, 7 * 8.0),
    ([16.] + [0.125] * 7, [16.] + [0.0625] * 7, 7 * 2.0 ** -5),  # e = 8
    ([16.] + [0.25] * 7, [16.] + [0.125] * 7, 0.0)])
def test_one_group(xs, ws, loss):
    import qwen_fastpath as qf
    x, w, s = _one_block(xs, ws)
    y = qf.fp8_w8a8_mm(x, w.t(), s, F32)
    want = sum(a * b for a, b in zip(xs, ws))
    assert (y.double() - want).abs().max().item() <= loss
    # the same small products in the next group, where nothing large stands beside them, are whole
    x, w, s = _one_block([xs[0]] + [0.] * 7 + xs[1:], [ws[0]] + [0.] * 7 + ws[1:])
    if xs[1] > 0:
        assert (qf.fp8_w8a8_mm(x, w.t(), s, F32).double() == want).all()
