"""Prompt chunks over the 4-bit cache whose row tiles fill the machine, so that no positions are split and workgroups run in the
order of the row tiles over all heads; against 64 bits.  Rows of a tile: 256, and 128 at D = 256."""
import pytest
import torch

import kv4_helpers as H
from test_gpu_kv4_attention import _batch, _call, _check

pytestmark = pytest.mark.gpu


def _unsplit(q, heads, kv, D):
    """More than half of the compute units have a row tile of a kv head, of requests of more than 64 rows."""
    rows, group = 128 if D == 256 else 256, heads // kv
    tiles = sum(-(-n * group // rows) for n in q if n * group > 64) * kv
    return tiles > torch.cuda.get_device_properties(0).multi_processor_count // 2


# kv heads that are a multiple of 8, which the order of workgroups gives an XCD each, and that are not; the last row tile partial
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("D,q,seq,heads,kv", [
    (64, 520, 700, 64, 8), (64, 1301, 1400, 45, 5), (64, 2403, 2403, 15, 3), (128, 517, 600, 64, 8), (128, 700, 701, 60, 10),
    (128, 1999, 2100, 21, 3), (256, 290, 400, 64, 8), (256, 515, 515, 35, 7)])
def test_one_chunk(D, q, seq, heads, kv, ragged):
    assert _unsplit([q], heads, kv, D)
    s = _batch(D + q, [seq], [q], heads, kv, D, 16)
    _check(s, _call(s, ragged=ragged))


@pytest.mark.parametrize("D,heads,kv,page", [(64, 16, 8, 16), (64, 10, 5, 48), (128, 24, 8, 64), (256, 18, 6, 16)])
def test_chunks_of_many_lengths(D, heads, kv, page):
    """Up to 64 requests, which go by their lengths, some of them short enough for the other kernel, or idle, or without positions."""
    g = H.gen(D)
    q = [int(torch.randint(60, 300, (1,), generator=g)) for _ in range(24)]
    q[3], q[4], q[11], q[17] = 0, 1, 7, 700
    seq = [n + int(torch.randint(0, 200, (1,), generator=g)) for n in q]
    seq[5], seq[6] = 0, q[6] // 2  # no positions; fewer than its tokens
    assert _unsplit(q, heads, kv, D)
    s = _batch(D + heads, seq, q, heads, kv, D, page)
    _check(s, _call(s))


@pytest.mark.parametrize("D,heads,kv", [(64, 20, 5), (64, 32, 8), (128, 12, 3), (256, 16, 4)])
@pytest.mark.parametrize("ragged", [False, True])
def test_more_requests_than_lanes(D, heads, kv, ragged):
    """More than 64 requests, which go in the order that they are given in."""
    g = H.gen(heads)
    n = 131
    q = [int(torch.randint(17, 60, (1,), generator=g)) for _ in range(n)] if ragged else [23] * n
    if ragged:
        q[0], q[64], q[70], q[130] = 0, 150, 2, 1
    seq = [max(0, m + int(torch.randint(-20, 90, (1,), generator=g))) for m in q]
    assert _unsplit(q, heads, kv, D)
    s = _batch(n + D, seq, q, heads, kv, D, 16)
    _check(s, _call(s))
