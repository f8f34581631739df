"""Norms of query and key heads with the rotation and the write into pages, against 64 bits: bounds from kv4_helpers, equality
for what goes into 4 bits."""
import pytest
import torch

import kv4_helpers as H
import qwen_fastpath as qf

pytestmark = pytest.mark.gpu
BF16, U8 = torch.bfloat16, torch.uint8


def _case(seed, T, heads, kv, D, rot, table=BF16, wide=1, norm=True, offset=0.0, positions=5000):
    g = H.gen(seed)
    qkv = torch.randn(T, (wide * heads + 2 * kv) * D, generator=g) * torch.exp(torch.randn(T, 1, generator=g))
    qkv[:, ::23] *= 10
    qkv = qkv.to(BF16)
    angle = torch.rand(positions, rot // 2, generator=g) * 6.3
    return dict(qkv=qkv, split=[wide * heads * D, kv * D, kv * D], sizes=(T, heads, kv, D), wide=wide,
                table=torch.cat([angle.cos(), angle.sin()], -1).to(table), positions=torch.randint(0, positions, (T,), generator=g),
                weights=[(1 - offset + 0.3 * torch.randn(D, generator=g)).to(BF16) for _ in range(2)] if norm else [None, None],
                offset=offset)


def _views(c, qkv):
    T, heads, kv, D = c["sizes"]
    q, k, v = qkv.split(c["split"], -1)
    return q.view(T, heads, -1)[..., :D], k.view(T, kv, D), v.view(T, kv, D)


def _want(c, interleaved, eps=1e-6):
    q, k, v = _views(c, c["qkv"])
    return [H.norm_rope(x, w, c["offset"], eps, c["table"], c["positions"], interleaved) for x, w in zip((q, k), c["weights"])] + [v]


def _gpu(t):
    return None if t is None else t.cuda()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,heads,kv,D,rot,table,wide,norm,offset", [
    (1, 1, 1, 64, 64, BF16, 1, True, 0.0), (3, 5, 1, 64, 16, BF16, 2, True, 1.0), (17, 6, 3, 64, 32, torch.float32, 1, False, 0.0),
    (1, 64, 8, 128, 128, BF16, 1, True, 0.0), (5, 8, 2, 128, 96, BF16, 1, True, 0.0), (33, 7, 7, 128, 48, torch.float32, 2, True, 1.0),
    (2, 3, 1, 256, 64, BF16, 2, True, 1.0), (9, 24, 4, 256, 256, torch.float32, 1, True, 0.0), (129, 2, 2, 256, 160, BF16, 1, True, 0.0),
    (700, 16, 2, 128, 64, BF16, 1, True, 0.0)])
def test_against_64_bits(T, heads, kv, D, rot, table, wide, norm, offset, interleaved):
    c = _case(T + D + rot, T, heads, kv, D, rot, table, wide, norm, offset)
    (q, q_slack), (k, k_slack), v = _want(c, interleaved)
    args = [*_views(c, c["qkv"].cuda())[:2], c["positions"].cuda(), c["table"].cuda(), *map(_gpu, c["weights"])]
    kw = dict(weight_offset=offset, interleaved=interleaved)
    got_q, got_k = qf.qk_norm_rope(*args, **kw)
    H.near(got_q, q, q_slack, "query")
    H.near(got_k, k, k_slack, "key")

    # into bf16 pages and into 4 bits, with tokens that have no slot; whatever else the pages hold stays
    g = H.gen(T)
    page = 16 if T < 100 else 64
    blocks = -(-T // page) + 1
    slots = torch.randperm(blocks * page, generator=g)[:T]
    if T > 2:
        slots[1], slots[T - 1] = -1, blocks * page
    on = (slots >= 0) & (slots < blocks * page)
    value = _views(c, c["qkv"].cuda())[2]
    pages = [torch.full((blocks, page, kv, D), 7.0, dtype=BF16, device="cuda") for _ in range(2)]
    q2, k2 = qf.qk_norm_rope(*args, value=value, cache=tuple(pages), slots=slots.cuda(), **kw)
    assert k2 is None and torch.equal(q2, got_q)
    for p, want in zip(pages, (got_k.cpu(), v)):
        all_ = torch.full((blocks * page, kv, D), 7.0, dtype=BF16)
        all_[slots[on]] = want[on]
        assert torch.equal(p.cpu().view(-1, kv, D), all_)

    cache = torch.zeros(blocks, kv, page // 16, 17 * D, dtype=U8, device="cuda")
    key_out = torch.empty(T, kv, D, dtype=BF16, device="cuda")
    q3, k3 = qf.qk_norm_rope(*args, value=value, cache=cache, slots=slots.cuda(), key_out=key_out, **kw)
    assert k3 is key_out and torch.equal(q3, got_q)
    exact = k.float().to(BF16)  # computed in 64 bits there: equal
    assert torch.equal(key_out.cpu(), exact)
    want_cache = torch.zeros_like(cache, device="cpu")
    H.write(want_cache, slots, exact, v)
    got = qf.kv4_load(cache, slots.cuda())
    for x, y in zip(got, (exact, v)):
        assert torch.equal(x.cpu().double(), torch.where(on[:, None, None], H.rounded(y), 0.0))
    assert torch.equal(cache.cpu()[..., 16 * D:], want_cache[..., 16 * D:])


def test_in_place_and_given_outputs():
    c = _case(1, 11, 4, 2, 128, 64)
    want_q, want_k = qf.qk_norm_rope(*_views(c, c["qkv"].cuda())[:2], c["positions"].cuda(), c["table"].cuda(), *map(_gpu, c["weights"]))
    qkv = c["qkv"].cuda()
    q, k, v = _views(c, qkv)
    a, b = qf.qk_norm_rope(q, k, c["positions"].cuda(), c["table"].cuda(), *map(_gpu, c["weights"]), query_out=q, key_out=k)
    assert a is q and b is k and torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(v.cpu(), _views(c, c["qkv"])[2])
    wide = torch.zeros(11, 6, 136, dtype=BF16, device="cuda")
    q, k, _ = _views(c, c["qkv"].cuda())
    out = wide[:, 1:5, :128]
    a, b = qf.qk_norm_rope(q, k, c["positions"].cuda(), c["table"].cuda(), *map(_gpu, c["weights"]), query_out=out)
    assert a is out and torch.equal(out, want_q) and not wide[:, 0].any() and not wide[:, 5].any() and not wide[:, :, 128:].any()


def test_without_rotation_and_with_one_norm():
    c = _case(2, 6, 3, 1, 64, 16)
    q, k, _ = _views(c, c["qkv"].cuda())
    a, b = qf.qk_norm_rope(q, k, None, None, c["weights"][0].cuda(), None)
    want, slack = H.norm_rope(_views(c, c["qkv"])[0], c["weights"][0], 0.0, 1e-6, None, None, False)
    H.near(a, want, slack)
    assert torch.equal(b, k)


def test_positions_are_kept_inside_the_table():
    c = _case(3, 4, 2, 1, 64, 64, positions=10)
    at = torch.tensor([-5, 10, 2 ** 40, 9])
    q, k, _ = _views(c, c["qkv"].cuda())
    a = qf.qk_norm_rope(q, k, at.cuda(), c["table"].cuda())[0]
    b = qf.qk_norm_rope(q, k, at.clamp(0, 9).cuda(), c["table"].cuda())[0]
    assert torch.equal(a, b)


def test_rows_of_zeros_infinities_and_nan():
    c = _case(4, 8, 2, 2, 128, 128)
    x = c["qkv"]
    x[1] = 0
    x[2, 3] = float("inf")
    x[3, 130] = float("nan")
    x[4] = 2.0 ** -70   # squares below the normal numbers
    x[5, :4] = 2.0 ** 60
    (q, q_slack), (k, _), _ = _want(c, False)
    got_q, got_k = qf.qk_norm_rope(*_views(c, x.cuda())[:2], c["positions"].cuda(), c["table"].cuda(), *map(_gpu, c["weights"]))
    rows = [0, 1, 4, 5, 6, 7]
    H.near(got_q[rows], q[rows], q_slack[rows])
    assert got_q[2, 0].isnan().any() and torch.equal(got_q[2, 1].cpu().isnan(), torch.zeros(128, dtype=torch.bool))
    assert got_q[3, 1].isnan().all() and not got_q[3, 0].isnan().any()
    assert not got_q[1].any()


def test_rows_whose_squares_leave_fp32():
    """Norms of values from 2^-120 to 2^120, without an eps that would hide the small ones."""
    c = _case(7, 13, 2, 2, 128, 64)
    x = (torch.randn(13, 6 * 128, generator=H.gen(1)) * torch.exp2(torch.arange(-120, 121, 20).double()[:, None])).to(BF16)
    c["qkv"] = x
    (q, q_slack), (k, k_slack), _ = _want(c, False, eps=0.0)
    a, b = qf.qk_norm_rope(*_views(c, x.cuda())[:2], c["positions"].cuda(), c["table"].cuda(), *map(_gpu, c["weights"]), eps=0.0)
    H.near(a, q, q_slack)
    H.near(b, k, k_slack)


@pytest.mark.parametrize("cache", ["pages", "kv4"])
def test_strided_pages(cache):
    """Pages interleaved key by value (bf16), and one layer of several (4 bits)."""
    c = _case(5, 20, 4, 2, 64, 32)
    slots = torch.arange(20)
    q, k, v = _views(c, c["qkv"].cuda())
    rest = (c["positions"].cuda(), c["table"].cuda(), *map(_gpu, c["weights"]))
    plain = qf.qk_norm_rope(q, k, *rest)[1]
    if cache == "pages":
        both = torch.zeros(2, 2, 16, 128, dtype=BF16, device="cuda")  # [blocks, heads, page, key then value]
        kp, vp = both[..., :64].transpose(1, 2), both[..., 64:].transpose(1, 2)
        qf.qk_norm_rope(q, k, *rest, value=v, cache=(kp, vp), slots=slots.cuda())
        assert torch.equal(kp.reshape(32, 2, 64)[:20], plain) and torch.equal(vp.reshape(32, 2, 64)[:20], v)
        assert not kp.reshape(32, 2, 64)[20:].any()
    else:
        layers = torch.zeros(2, 3, 2, 1, 17 * 64, dtype=U8, device="cuda")
        one = qf.kv4_cache(2, 16, 2, 64)
        qf.qk_norm_rope(q, k, *rest, value=v, cache=layers[:, 2], slots=slots.cuda())
        qf.qk_norm_rope(q, k, *rest, value=v, cache=one, slots=slots.cuda())
        assert torch.equal(layers[:, 2], one) and not layers[:, :2].any() and one.any()


def test_a_token_alone_and_in_a_batch():
    """A token's bits do not depend on what else the call holds."""
    c = _case(6, 40, 8, 2, 128, 128)
    q, k, v = _views(c, c["qkv"].cuda())
    rest = (c["table"].cuda(), *map(_gpu, c["weights"]))
    all_, one = qf.kv4_cache(3, 16, 2, 128), qf.kv4_cache(3, 16, 2, 128)
    slots = torch.arange(40).cuda()
    together = qf.qk_norm_rope(q, k, c["positions"].cuda(), *rest, value=v, cache=all_, slots=slots)[0]
    for t in range(40):
        a = qf.qk_norm_rope(q[t:t + 1], k[t:t + 1], c["positions"][t:t + 1].cuda(), *rest, value=v[t:t + 1], cache=one,
                            slots=slots[t:t + 1])[0]
        assert torch.equal(a[0], together[t])
    assert torch.equal(all_, one)
