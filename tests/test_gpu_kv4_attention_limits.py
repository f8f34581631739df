"""Attention over the 4-bit cache at the longest sequence that a table may name: 2^31 - 64 positions, all of them one block's."""
import pytest
import torch

import qwen_fastpath as qf

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
MOST = 2 ** 31 - 64


@pytest.mark.parametrize("q", [2, 65])
def test_the_longest_sequence(q):
    """Keys of 0 and values of 1: each weight is 1, sums of them are whole numbers that fp32 holds but for their ends (2^-24), and
    an output is 1.  65 tokens take the kernel of many rows, which asks for places ahead of its last stage."""
    D = 64
    cache = qf.kv4_cache(1, 16, 1, D)
    qf.kv4_store(torch.zeros(16, 1, D, dtype=BF16, device="cuda"), torch.ones(16, 1, D, dtype=BF16, device="cuda"), cache,
                 torch.arange(16, device="cuda"))
    table = torch.zeros(1, MOST // 16, dtype=I32, device="cuda")
    query = torch.randn(q, 1, D, generator=torch.Generator().manual_seed(q)).to(BF16).cuda()
    for seq in (MOST, MOST - 63):
        print(f"{q} tokens of {seq}", flush=True)
        got = qf.kv4_attention(query, cache, torch.tensor([seq], dtype=I32, device="cuda"), table, 0.125, q_len=q)
        assert bool((got == 1).all())
