"""The fused norms, gate and residual on the GPU against 64 bits, with derived bounds."""
import itertools

import pytest
import torch

import block_helpers as H

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def qf():
    import qwen_fastpath
    return qwen_fastpath


def _inputs(M, N, wide, gate, seed):
    g = H.gen(seed)
    x = H.rows(g, M, N)
    r = 4 * torch.randn(M, N, generator=g)
    shape = {"none": None, "channel": (N,), "token": (M, 1), "full": (M, N)}[gate]
    return (x, r if wide else r.to(BF16), (1 + 0.2 * torch.randn(N, generator=g)).to(BF16),
            (1 + 0.2 * torch.randn(N, generator=g)).to(BF16),
            None if shape is None else (2 * torch.randn(*shape, generator=g)).to(BF16))


# A row's sum of squares in fp32: a thread adds at most 32 of them, 6 exchanges and at most 16 wavefronts follow, so no
# term takes part in more than 54 additions and the sum is off by at most 55 * 2^-24 (the square's rounding among them);
# its root halves that, the root, the reciprocal, the division and eps add 2^-24 each.  With the factors' roundings:
ROW = 40 * 2.0 ** -24


def _reference(x, r, post, pre, gate, act, alpha, eps, offset):
    """(y, h, bounds before their last rounding)"""
    p, rel = x.double(), 0.0
    if post is not None:
        p = p / torch.sqrt(p.pow(2).mean(1, keepdim=True) + eps) * (offset + post.double())
        rel = ROW
    if gate is not None:
        g = gate.double()
        if act == "sigmoid":
            # exp2 of a rounded product: |g| log2(e) 2^-24 ln 2 and two steps; then the sum and the reciprocal
            p, rel = p * torch.sigmoid(g), rel + (g.abs() + 8) * 2.0 ** -23
        else:
            p = p * g
    add = alpha * p
    y = r.double() + add
    bound = add.abs() * (rel + 8 * H.F32) + y.abs() * 2 * H.F32
    scale = 1 / torch.sqrt(y.pow(2).mean(1, keepdim=True) + eps)
    w = 1.0 if pre is None else offset + pre.double()
    h = y * scale * w
    # y's errors move the row's mean square by at most 2 |y| bound / N in all: half of that moves the norm
    moved = (y.abs() * bound).mean(1, keepdim=True) * scale ** 2
    return y, h, bound, (bound * scale * w.abs() if pre is not None else bound * scale) + h.abs() * (ROW + moved)


def _check(qf, M, N, wide=False, post=True, pre=True, gate="none", act="none", alpha=0.7, eps=1e-6, offset=0.0, seed=0):
    x, r, wp, wq, g = _inputs(M, N, wide, gate, seed)
    wp, wq = wp if post else None, wq if pre else None
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    y, h = qf.block_norm_rows(dev(x), dev(r), dev(wp), dev(wq), gate=dev(g), gate_act=act, alpha=alpha, eps=eps,
                              weight_offset=offset)
    torch.cuda.synchronize()
    assert y.dtype == (F32 if wide else BF16) and h.dtype == BF16
    ry, rh, by, bh = _reference(x, r, wp, wq, g, act, alpha, eps, offset)
    H.within(y, ry, by, H.F32 if wide else H.BF16)
    H.within(h, rh, bh, H.BF16)


@pytest.mark.parametrize("M,N", [(1, 8), (3, 64), (17, 128), (33, 136), (5, 512), (4, 520), (1, 5120), (7, 2568), (2, 8192),
                                 (3, 8200), (2, 16384), (2, 16392), (1, 32768), (1000, 96)])
@pytest.mark.parametrize("wide", [False, True])
def test_sizes(qf, M, N, wide):
    _check(qf, M, N, wide, gate="full", act="sigmoid", seed=N)
    _check(qf, M, N, wide, seed=N + 1)


@pytest.mark.parametrize("gate,act,post,pre,wide", list(itertools.product(
    ["none", "channel", "token", "full"], ["none", "sigmoid"], [False, True], [False, True], [False, True])))
def test_forms(qf, gate, act, post, pre, wide):
    _check(qf, 5, 648, wide, post, pre, gate, act, alpha=-1.25, offset=1.0, seed=3)


def test_zero_rows_and_extremes(qf):
    x = torch.zeros(4, 640, dtype=BF16)
    r = torch.zeros(4, 640, dtype=BF16)
    x[1] = 1e18  # squares far from fp32's ends
    r[2] = float("inf")
    x[3, 5] = float("nan")
    w = torch.ones(640, dtype=BF16)
    y, h = qf.block_norm_rows(x.cuda(), r.cuda(), w.cuda(), w.cuda(), eps=0.0 + 1e-6)
    y, h = y.cpu().float(), h.cpu().float()
    assert y[0].eq(0).all() and h[0].eq(0).all()
    assert (y[1] - 1).abs().max() <= H.BF16 and (h[1] - 1).abs().max() <= 2 * H.BF16
    assert torch.isinf(y[2]).all() and torch.isnan(h[2]).all()
    assert torch.isnan(y[3]).all() and torch.isnan(h[3]).all()


@pytest.mark.parametrize("M,N,wide", [(9, 5120, False), (9, 96, True), (9, 16392, True)])
def test_in_place_and_strided(qf, M, N, wide):
    x, r, wp, wq, g = (None if t is None else t.cuda() for t in _inputs(M, N, wide, "full", 2))
    kw = dict(gate=g, gate_act="sigmoid", alpha=0.5)
    y, h = qf.block_norm_rows(x, r, wp, wq, **kw)
    wide_x = torch.zeros(M, N + 24, dtype=BF16, device="cuda")
    wide_r = torch.zeros(M, N + 40, dtype=r.dtype, device="cuda")
    xv, rv = wide_x[:, 8:N + 8], wide_r[:, 8:N + 8]
    xv.copy_(x), rv.copy_(r)
    y2, h2 = qf.block_norm_rows(xv, rv, wp, wq, **kw)
    assert torch.equal(y2, y) and torch.equal(h2, h)
    odd = torch.zeros(M, N + 5, dtype=BF16, device="cuda")
    odd[:, 3:N + 3] = x
    y2, h2 = qf.block_norm_rows(odd[:, 3:N + 3], r, wp, wq, **kw)
    assert torch.equal(y2, y) and torch.equal(h2, h)
    gate = g.t().contiguous().t()
    y2, h2 = qf.block_norm_rows(x, r, wp, wq, gate=gate, gate_act="sigmoid", alpha=0.5)
    assert torch.equal(y2, y) and torch.equal(h2, h)
    y3, h3 = qf.block_norm_rows(xv, rv, wp, wq, y=rv, h=xv, **kw)  # in place
    assert y3 is rv and h3 is xv and torch.equal(rv, y) and torch.equal(xv, h)
    assert wide_x[:, :8].eq(0).all() and wide_x[:, N + 8:].eq(0).all()
    assert wide_r[:, :8].eq(0).all() and wide_r[:, N + 8:].eq(0).all()


def test_broadcast_gates(qf):
    x, r, wp, wq, g = (None if t is None else t.cuda() for t in _inputs(6, 640, False, "channel", 4))
    y, h = qf.block_norm_rows(x, r, wp, wq, gate=g)
    y2, h2 = qf.block_norm_rows(x, r, wp, wq, gate=g.expand(6, 640))
    assert torch.equal(y, y2) and torch.equal(h, h2)
    t = torch.randn(1, 1, device="cuda").to(BF16)
    y, h = qf.block_norm_rows(x, r, wp, wq, gate=t.expand(6, 1))
    y2, h2 = qf.block_norm_rows(x, r, wp, wq, gate=t.expand(6, 640))
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_no_rows(qf):
    x = torch.zeros(0, 64, dtype=BF16, device="cuda")
    y, h = qf.block_norm_rows(x, x.float())
    assert y.shape == (0, 64) and y.dtype == F32 and h.shape == (0, 64)


def test_graph_replays(qf):
    x, r, wp, wq, g = (None if t is None else t.cuda() for t in _inputs(5, 5120, False, "token", 6))
    want = qf.block_norm_rows(x, r, wp, wq, gate=g)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    sx = torch.zeros_like(x)
    with torch.cuda.graph(graph, stream=stream):
        y, h = qf.block_norm_rows(sx, r, wp, wq, gate=g)
    for v in (x, torch.zeros_like(x), x):
        sx.copy_(v)
        graph.replay()
        ref = qf.block_norm_rows(v, r, wp, wq, gate=g)
        torch.cuda.synchronize()
        assert torch.equal(y, ref[0]) and torch.equal(h, ref[1])
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])


def test_plain_calls_agree_with_the_long_way(qf, monkeypatch):
    import qwen_fastpath._qf_block_call as plain
    g = H.gen(5)
    x, r = torch.randn(9, 520, generator=g).to(BF16).cuda(), torch.randn(9, 520, generator=g).cuda()
    w = torch.randn(520, generator=g).to(BF16).cuda()
    calls = [lambda r=r, gate=gate, act=act: qf.block_norm_rows(x, r, w, None, gate, act, 0.5, 1e-5, 1.0)
             for r in (r, r.to(BF16)) for gate in (None, w, x[:, :1], x) for act in ("none", "sigmoid")]
    took = []
    real = plain.norm
    monkeypatch.setattr(plain, "norm", lambda *a: took.append(real(*a)) or took[-1])
    short = [f() for f in calls]
    assert len(took) == len(calls) and all(t is not None for t in took)
    monkeypatch.setattr(plain, "norm", lambda *a: None)
    for a, f in zip(short, calls):
        b = f()
        assert a[0].dtype == b[0].dtype and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_wrong_calls_on_the_gpu(qf):
    x = torch.zeros(4, 64, dtype=BF16, device="cuda")
    for f in (lambda: qf.block_norm_rows(x.half(), x), lambda: qf.block_norm_rows(x, x.half()), lambda: qf.block_norm_rows(x, x, x[0].float()),
              lambda: qf.block_norm_rows(x, x, None, x[0, :32]), lambda: qf.block_norm_rows(x, x, gate=x[0].float())):
        with pytest.raises(TypeError):
            f()
    for f in (lambda: qf.block_norm_rows(x, x[:3]), lambda: qf.block_norm_rows(x[:, :60].contiguous(), x[:, :60].contiguous()),
              lambda: qf.block_norm_rows(x, x, gate=x[:, :2]), lambda: qf.block_norm_rows(x, x, gate=x[0, :4]),
              lambda: qf.block_norm_rows(x, x, gate_act="silu"), lambda: qf.block_norm_rows(x, x, eps=-1.0),
              lambda: qf.block_norm_rows(x, x.cpu())):
        with pytest.raises(ValueError):
            f()
