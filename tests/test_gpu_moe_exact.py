"""The experts' layer with integers, bit for bit (exact_cases): the activation's 16 bits, every unit and block of the sums."""
import pytest
import torch

import block_helpers as H
import exact_cases as X

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,k,Hd,I", X.MOE)
def test_layer(T, E, k, Hd, I):
    import qwen_fastpath as qf
    x, logits, up, down, chosen = X.experts(T, E, k, Hd, I)
    want = X.layer(X.layer_units(x, up, down, chosen), T, Hd)
    image = lambda ws: qf.fp8_to_tiled(torch.cat([q.view(torch.uint8) for q, _ in ws]).view(H.FP8).cuda().t())  # noqa: E731
    args = (image(up), torch.stack([s for _, s in up]).cuda(), image(down), torch.stack([s for _, s in down]).cuda(), k)
    for renormalize in (True, False):  # the other logits are -inf: the same weights
        for l in (logits, logits.to(torch.bfloat16)):
            y = qf.moe_few_tokens(x.cuda(), l.cuda(), *args, renormalize=renormalize).cpu()
            wrong = (y != want).nonzero()
            assert not len(wrong), f"{len(wrong)} of {y.numel()} values differ, the first at {wrong[0].tolist()}"
