"""Norms of query and key heads with the rotation where a wavefront takes several rows one after the other (many tokens), and
rows whose squares fp32 does not hold, against 64 bits."""
import pytest
import torch

import kv4_helpers as H
import qwen_fastpath as qf

pytestmark = pytest.mark.gpu
BF16, U8 = torch.bfloat16, torch.uint8


def _inputs(seed, T, heads, kv, D, rot, table):
    g = H.gen(seed)
    x = [(torch.randn(T, n, D, generator=g) * torch.exp(torch.randn(T, n, 1, generator=g))).to(BF16) for n in (heads, kv, kv)]
    angle = torch.rand(900, rot // 2, generator=g) * 6.3
    weights = [(1 + 0.3 * torch.randn(D, generator=g)).to(BF16) for _ in range(2)]
    return x, torch.cat([angle.cos(), angle.sin()], -1).to(table), torch.randint(0, 900, (T,), generator=g), weights


# 2 to 4 rows a lane; heads and tokens that end inside a wavefront's share
@pytest.mark.parametrize("T,heads,kv,D,rot,table,interleaved", [
    (1500, 17, 5, 64, 48, torch.float32, False), (1203, 33, 3, 128, 128, BF16, False), (1203, 33, 3, 128, 64, BF16, True),
    (530, 24, 4, 256, 64, torch.float32, False), (2049, 4, 1, 256, 256, BF16, True)])
def test_many_tokens(T, heads, kv, D, rot, table, interleaved):
    (q, k, v), cs, positions, weights = _inputs(T + D, T, heads, kv, D, rot, table)
    (want_q, q_slack), (want_k, k_slack) = (H.norm_rope(x, w, 0.0, 1e-6, cs, positions, interleaved) for x, w in zip((q, k), weights))
    page, blocks = 48, -(-T // 48) + 1
    slots = torch.arange(T) + 5  # as a prompt's: neighbours, but not from a page's start
    slots[7], slots[T - 1] = -1, blocks * page
    on = slots >= 0
    on[T - 1] = False
    args = [t.cuda() for t in (q, k, positions, cs, *weights)]
    for pages in (False, True):
        if pages:
            cache = tuple(torch.full((blocks, page, kv, D), 7.0, dtype=BF16, device="cuda") for _ in range(2))
        else:
            cache = torch.zeros(blocks, kv, page // 16, 17 * D, dtype=U8, device="cuda")
        key_out = torch.empty(T, kv, D, dtype=BF16, device="cuda")
        got_q, _ = qf.qk_norm_rope(*args, value=v.cuda(), cache=cache, slots=slots.cuda(), key_out=key_out, interleaved=interleaved)
        H.near(got_q, want_q, q_slack, "query")
        if pages:
            H.near(key_out, want_k, k_slack, "key")
            for p, want in zip(cache, (key_out.cpu(), v)):
                all_ = torch.full((blocks * page, kv, D), 7.0, dtype=BF16)
                all_[slots[on]] = want[on]
                assert torch.equal(p.cpu().view(-1, kv, D), all_)
        else:
            exact = want_k.float().to(BF16)
            assert torch.equal(key_out.cpu(), exact)
            for got, want in zip(qf.kv4_load(cache, slots.cuda()), (exact, v)):
                assert torch.equal(got.cpu().double(), torch.where(on[:, None, None], H.rounded(want), 0.0))


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -120, 2.0 ** -105, 1e-6, 2.0 ** 100])
@pytest.mark.parametrize("D,interleaved", [(64, True), (128, True), (256, False)])
def test_rows_from_the_smallest_to_the_largest(D, interleaved, eps):
    """Rows of 2^-130 to 2^122 beside each other (D = 64: 8 of a wavefront), those that fp32's squares hold among them."""
    (q, k, _), cs, positions, weights = _inputs(D, 19, 3, 2, D, 32, torch.float32)
    scale = torch.exp2(torch.arange(-130, 123, 14).double())[:, None, None]
    q, k = ((x.double() / x.double().abs().amax(-1, keepdim=True) * scale).to(BF16) for x in (q, k))
    got = qf.qk_norm_rope(*(t.cuda() for t in (q, k, positions, cs, *weights)), eps=eps, interleaved=interleaved)
    for y, x, w in zip(got, (q, k), weights):
        want, slack = H.norm_rope(x, w, 0.0, eps, cs, positions, interleaved)
        H.near(y, want, slack)


def test_a_row_outside_the_rotation_keeps_its_bits():
    """Without norms and behind rot a value is passed on, the sign of a zero and an infinity among them."""
    (q, k, _), cs, positions, _ = _inputs(3, 21, 3, 2, 128, 32, BF16)
    q[:, :, 40], q[:, :, 41], q[:, :, 42] = -0.0, float("inf"), -float("inf")
    a, b = qf.qk_norm_rope(q.cuda(), k.cuda(), positions.cuda(), cs.cuda())
    for y, x in ((a, q), (b, k)):
        assert torch.equal(y.cpu()[..., 32:].view(torch.int16), x[..., 32:].view(torch.int16))
