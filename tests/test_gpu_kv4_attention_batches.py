"""Attention over the 4-bit cache where the batch or the tables decide how it is launched: many requests over many heads, long
tables, the join's two forms; against 64 bits."""
import pytest
import torch

import kv4_helpers as H
from test_gpu_kv4_attention import _batch, _call, _check

pytestmark = pytest.mark.gpu


def _lengths(seed, n, most):
    g = H.gen(seed)
    return [int(torch.randint(1, most, (1,), generator=g)) for _ in range(n)]


# requests * kv heads from 256 on: several workgroups a compute unit (few rows), or one (many registers, over 128 requests)
@pytest.mark.parametrize("B,q,heads,kv,D", [
    (40, 1, 16, 8, 128), (33, 2, 16, 8, 64), (33, 6, 24, 8, 64), (36, 5, 32, 8, 128), (65, 1, 8, 4, 256), (64, 5, 16, 4, 256), (131, 1, 4, 2, 128)])
def test_requests_that_fill_the_machine(B, q, heads, kv, D):
    seq = _lengths(B + D, B, 700)
    seq[3], seq[7] = 2500, 0
    s = _batch(B, seq, [q] * B, heads, kv, D, 16)
    _check(s, _call(s))


@pytest.mark.parametrize("seq,q,heads,kv,D", [
    ([4500], 1, 8, 8, 128), ([4100, 9], 3, 8, 4, 64), ([6000], 2, 12, 4, 256), ([5000], 6, 8, 2, 128), ([300, 1, 0, 2], 1, 4, 2, 128)])
def test_tables_wider_than_any_request(seq, q, heads, kv, D):
    """Rows of a table that could hold far more than the requests do, as a server's are: their other entries are out of range."""
    s = _batch(sum(seq) + D, seq, [q] * len(seq), heads, kv, D, 16)
    wide = torch.full((len(seq), 2048), -7, dtype=torch.int32)
    wide[:, :s["table"].shape[1]] = s["table"]
    want = _call(s)
    s["table"] = wide
    got = _call(s)
    _check(s, got)
    assert torch.equal(got, want)  # the launch differs, not what it computes


def test_a_wide_table_after_a_narrow_one():
    """The same kernel with less and with more LDS, in either order."""
    for widths in ((300, 64, 300), (64, 300)):
        for w in widths:
            s = _batch(w, [900], [1], 4, 2, 128, 16)
            wide = torch.zeros(1, w, dtype=torch.int32)
            wide[:, :s["table"].shape[1]] = s["table"]
            s["table"] = wide
            _check(s, _call(s))


@pytest.mark.parametrize("B,D", [(7, 128), (7, 256), (64, 64), (70, 64)])
def test_chunks_in_any_order(B, D):
    """Requests of equal and of different lengths, the longest last, some that only single tokens have, some with none."""
    g = H.gen(B + D)
    seq = sorted(_lengths(D, B, 260))
    seq[1] = seq[2] = seq[3]
    q = [int(torch.randint(0, 60, (1,), generator=g)) for _ in range(B)]
    q[0], q[B - 1], q[B - 2] = 0, 90, 1
    s = _batch(B * D, seq, q, 4, 2, D, 16)
    _check(s, _call(s))
    back = dict(s, seq=seq[::-1], q=q[::-1], cu=torch.tensor([0] + q[::-1]).cumsum(0), table=s["table"].flip(0), keys=s["keys"][::-1],
                vals=s["vals"][::-1])
    _check(back, _call(back))
