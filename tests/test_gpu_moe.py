"""The mixture-of-experts layer for a few tokens on the GPU against 64 bits, with derived bounds; and the operators of a
block-scaled layer run together."""
import pytest
import torch

import block_helpers as H

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")


@pytest.fixture(scope="module")
def qf():
    import qwen_fastpath
    return qwen_fastpath


def _layer(g, E, Hd, I):
    """Experts as ([2 I, H] q, s), ([H, I] q, s) each."""
    up, down = [], []
    for _ in range(E):
        (qg, sg), (qu, su) = H.weight(g, I, Hd), H.weight(g, I, Hd)
        up.append((torch.cat([qg.view(torch.uint8), qu.view(torch.uint8)]).view(H.FP8), torch.cat([sg, su])))
        down.append(H.weight(g, Hd, I))
    return up, down


def _on(qf, up, down):
    img = lambda ws: qf.fp8_to_tiled(torch.cat([q.view(torch.uint8) for q, _ in ws]).view(H.FP8).cuda().t())  # noqa: E731
    return img(up), torch.stack([s for _, s in up]).cuda(), img(down), torch.stack([s for _, s in down]).cuda()


def _routing(logits, k, renorm):
    """{token: [(expert, weight)]} from the definition, in 64 bits."""
    out = {}
    for t, row in enumerate(logits.double().tolist()):
        order = sorted(range(len(row)), key=lambda e: (-row[e] if row[e] == row[e] else -INF, e))
        chosen = order[:k]
        top = row[order[0]]
        if top == -INF:
            out[t] = []
            continue
        v = torch.tensor(row, dtype=torch.float64)
        e = torch.exp(v - v[order[0]])
        total = e[chosen].sum() if renorm else e.sum()
        out[t] = [(i, (e[i] / total).item()) for i in chosen if e[i] != 0]
    return out


def _reference(x, logits, up, down, k, renorm):
    T, Hd = x.shape
    I = down[0][0].shape[1]
    y = torch.zeros(T, Hd, dtype=torch.float64)
    bound = torch.zeros(T, Hd, dtype=torch.float64)
    for t, chosen in _routing(logits, k, renorm).items():
        for e, c in chosen:
            nb = H.blocks(I)
            q13, s13 = up[e]
            xd = x[t].double()
            ends = []
            for q, s in ((q13[:I], s13[:nb]), (q13[I:], s13[nb:])):
                w = H.widen(q, s)
                ends.append((w @ xd, (Hd + 8) * H.SUM * (w.abs() @ xd.abs())))
            (g, eg), (u, eu) = ends
            silu = g * torch.sigmoid(g)
            # the slope of silu is below 1.1; exp, the sum, the division and the product add a few roundings
            err = 1.1 * eg * (u.abs() + eu) + silu.abs() * eu + (silu * u).abs() * (g.abs() + 16) * 2.0 ** -23
            a = silu * u
            w2 = H.widen(*down[e])
            y[t] += c * (w2 @ a)
            # the activation as two bf16 numbers: what the first leaves (2^-8) is rounded by 2^-8 of itself; the sums, of
            # both; the weight c (its logits differ by at most 100: 100 * 2^-24 in the exponent, and the sum's and
            # quotient's roundings: 2^-16 covers them)
            bound[t] += c * (w2.abs() @ (err + 2.0 ** -16 * a.abs())) + c * (w2.abs() @ a.abs()) * (
                (2 * k * I + 16) * H.SUM + 2.0 ** -16)
    return y, bound


def _check(qf, T, E, k, Hd, I, renorm=True, dtype=F32, logits=None, seed=0):
    g = H.gen(seed)
    up, down = _layer(g, E, Hd, I)
    x = (torch.randn(T, Hd, generator=g)).to(BF16)
    if logits is None:
        logits = (2 * torch.randn(T, E, generator=g)).to(dtype)
    w = _on(qf, up, down)
    y = qf.moe_few_tokens(x.cuda(), logits.cuda(), *w, k, renormalize=renorm)
    torch.cuda.synchronize()
    ref, bound = _reference(x, logits, up, down, k, renorm)
    H.within(y, ref, bound, H.BF16)
    return x, logits, w, y


@pytest.mark.parametrize("T,E,k,Hd,I", [(1, 1, 1, 64, 64), (1, 8, 2, 128, 128), (2, 5, 5, 192, 64), (3, 60, 4, 320, 192),
                                        (16, 16, 8, 256, 128), (16, 4, 1, 64, 320), (7, 130, 16, 128, 64),
                                        (5, 512, 8, 64, 64), (16, 65, 3, 1088, 192), (4, 8, 8, 2112, 1344)])
@pytest.mark.parametrize("renorm", [True, False])
def test_sizes(qf, T, E, k, Hd, I, renorm):
    _check(qf, T, E, k, Hd, I, renorm, F32 if renorm else BF16, seed=T + E)


# output channels in one group of workgroups, in two splits, in none; an odd last tile; many units
@pytest.mark.parametrize("T,E,k,Hd,I", [(2, 3, 2, 4096, 64), (2, 3, 2, 4160, 64), (3, 4, 2, 8192, 192), (16, 40, 8, 2688, 448),
                                        (9, 20, 16, 64, 1344)])
def test_splits_of_the_second_product(qf, T, E, k, Hd, I):
    _check(qf, T, E, k, Hd, I, True, seed=Hd)


def test_plain_calls_agree_with_the_long_way(qf, monkeypatch):
    import qwen_fastpath._qf_block_call as plain
    g = H.gen(2)
    w = _on(qf, *_layer(g, 5, 128, 192))
    x, logits = torch.randn(7, 128, generator=g).to(BF16).cuda(), torch.randn(7, 5, generator=g).cuda()
    calls = [lambda T=T, l=l, n=n: qf.moe_few_tokens(x[:T], l[:T], *w, 3, n) for T in (1, 7) for l in (logits, logits.to(BF16)) for n in (True, False)]
    took = []
    real = plain.moe
    monkeypatch.setattr(plain, "moe", lambda *a: took.append(real(*a)) or took[-1])
    short = [f() for f in calls]
    assert len(took) == len(calls) and all(t is not None for t in took)
    monkeypatch.setattr(plain, "moe", lambda *a: None)
    assert all(torch.equal(a, f()) for a, f in zip(short, calls))


def test_wrong_calls_on_the_gpu(qf):
    g = H.gen(2)
    w13, s13, w2, s2 = _on(qf, *_layer(g, 5, 128, 192))
    x, logits = torch.zeros(7, 128, dtype=BF16, device="cuda"), torch.zeros(7, 5, device="cuda")
    for f in (lambda: qf.moe_few_tokens(x.half(), logits, w13, s13, w2, s2, 2), lambda: qf.moe_few_tokens(x, logits.half(), w13, s13, w2, s2, 2),
              lambda: qf.moe_few_tokens(x, logits, w13, s13.half(), w2, s2, 2)):
        with pytest.raises(TypeError):
            f()
    for f in (lambda: qf.moe_few_tokens(x, logits[:6], w13, s13, w2, s2, 2), lambda: qf.moe_few_tokens(x, logits, w13, s13, w2, s2, 0),
              lambda: qf.moe_few_tokens(x, logits, w13, s13, w2, s2, 6), lambda: qf.moe_few_tokens(x, logits[:, :4], w13, s13, w2, s2, 2),
              lambda: qf.moe_few_tokens(x, logits, w13, s13[:, :2], w2, s2, 2), lambda: qf.moe_few_tokens(x, logits, w13[:-1], s13, w2, s2, 2),
              lambda: qf.moe_few_tokens(x, logits, w13, s13, w2, s2.cpu(), 2),
              lambda: qf.moe_few_tokens(torch.cat([x, x, x]), torch.cat([logits, logits, logits]), w13, s13, w2, s2, 2)):
        with pytest.raises(ValueError):
            f()


def test_two_graphs_at_once(qf):
    g = H.gen(6)
    w = _on(qf, *_layer(g, 9, 512, 384))
    xs = [torch.randn(16, 512, generator=g).to(BF16).cuda() for _ in range(3)]
    logits = torch.randn(16, 9, generator=g).cuda()
    want = [qf.moe_few_tokens(x, logits, *w, 3) for x in xs]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for x in xs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(qf.moe_few_tokens(x, logits, *w, 3))
        graphs.append(graph)
    sides = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        for side, graph in zip(sides, graphs):
            with torch.cuda.stream(side):
                graph.replay()
        eager = qf.moe_few_tokens(xs[2], logits, *w, 3)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])


def test_every_token_count(qf):
    g = H.gen(11)
    up, down = _layer(g, 12, 128, 128)
    w = _on(qf, up, down)
    x = torch.randn(16, 128, generator=g).to(BF16)
    logits = torch.randn(16, 12, generator=g)
    for T in range(1, 17):
        y = qf.moe_few_tokens(x[:T].cuda(), logits[:T].cuda(), *w, 3)
        ref, bound = _reference(x[:T], logits[:T], up, down, 3, True)
        H.within(y, ref, bound, H.BF16)
    assert qf.moe_few_tokens(x[:0].cuda(), logits[:0].cuda(), *w, 3).shape == (0, 128)


def test_ties_take_the_lowest_index(qf):
    logits = torch.zeros(4, 70)
    logits[1, 3::2] = 1.0
    logits[2] = -0.0
    logits[2, ::2] = 0.0  # equal to -0
    logits[3] = torch.arange(70).flip(0) // 10
    _check(qf, 4, 70, 5, 64, 64, True, logits=logits, seed=1)
    _check(qf, 4, 70, 5, 64, 64, False, logits=logits.to(BF16), seed=2)


def test_masked_logits_and_empty_rows(qf):
    logits = torch.randn(6, 20, generator=H.gen(0))
    logits[0] = -INF                 # no expert at all
    logits[1, 1:] = -INF             # one, with k = 4
    logits[2, 5:] = -INF
    logits[3] = -3.0e38              # the type's low end: even weights
    logits[4, 7] = 200.0             # the others' weights vanish
    _, _, _, y = _check(qf, 6, 20, 4, 128, 64, True, logits=logits, seed=3)
    assert y[0].eq(0).all()
    logits[:] = -INF
    x, _, w, y = _check(qf, 6, 20, 4, 128, 64, False, logits=logits, seed=3)
    assert y.eq(0).all()


def test_nan_stays_with_its_token_and_expert(qf):
    g = H.gen(4)
    up, down = _layer(g, 6, 128, 64)
    x = torch.randn(4, 128, generator=g).to(BF16)
    logits = torch.full((4, 6), -INF)
    for t, e in ((0, 0), (0, 1), (1, 1), (1, 2), (2, 3), (2, 4), (3, 4), (3, 5)):
        logits[t, e] = 1.0 + t
    clean = qf.moe_few_tokens(x.cuda(), logits.cuda(), *_on(qf, up, down), 2)
    x2 = x.clone()
    x2[0, 7] = float("nan")
    y = qf.moe_few_tokens(x2.cuda(), logits.cuda(), *_on(qf, up, down), 2)
    assert torch.isnan(y[0]).all() and torch.equal(y[1:], clean[1:])
    down[4][0].view(torch.uint8)[:, 3] = 0x7f
    y = qf.moe_few_tokens(x.cuda(), logits.cuda(), *_on(qf, up, down), 2)
    assert torch.isnan(y[2:]).all() and torch.equal(y[:2], clean[:2])
    bad = logits.clone()
    bad[3, 5] = float("nan")  # NaN is the largest, and its softmax no number
    y = qf.moe_few_tokens(x.cuda(), bad.cuda(), *_on(qf, up, down), 2)
    assert torch.isnan(y[3]).all() and torch.equal(y[:2], clean[:2])


def test_strided_inputs(qf):
    x, logits, w, y = _check(qf, 5, 30, 4, 192, 128, seed=6)
    wide = torch.zeros(5, 211, dtype=BF16, device="cuda")
    wide[:, 3:195] = x.cuda()
    lw = torch.zeros(5, 64, device="cuda")
    lw[:, 7:37] = logits.cuda()
    assert torch.equal(qf.moe_few_tokens(wide[:, 3:195], lw[:, 7:37], *w, 4), y)
    assert torch.equal(qf.moe_few_tokens(x.cuda(), logits.cuda().t().contiguous().t(), *w, 4), y)


def test_graph_replays_with_other_routings(qf):
    x, logits, w, y = _check(qf, 6, 40, 4, 320, 192, seed=7)
    x = x.cuda()
    sl = logits.cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = qf.moe_few_tokens(x, sl, *w, 4)
    for seed in (0, 1, 2):
        l = torch.randn(6, 40, generator=H.gen(seed)).cuda()
        sl.copy_(l)
        graph.replay()
        ref = qf.moe_few_tokens(x, l, *w, 4)
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


def test_two_streams_at_once(qf):
    x, logits, w, y = _check(qf, 16, 64, 8, 256, 128, seed=8)
    x, logits = x.cuda(), logits.cuda()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(qf.moe_few_tokens(x, logits, *w, 8))
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o in got)


@pytest.mark.parametrize("T", [3, 16, 40])
def test_a_layer_of_them_together(qf, T):
    """norms -> projection -> norms -> experts (or, above 16 tokens, a dense down projection) -> norms, captured in a graph
    and replayed, against the same calls one by one, each checked by its own bound."""
    g = H.gen(T)
    Hd, I, E, k = 256, 128, 12, 3
    q, s = H.weight(g, Hd, Hd)
    up, down = _layer(g, E, Hd, I)
    wts = [(1 + 0.1 * torch.randn(Hd, generator=g)).to(BF16) for _ in range(4)]
    x0 = torch.randn(T, Hd, generator=g).to(BF16)
    r0 = torch.randn(T, Hd, generator=g).to(BF16)
    router = torch.randn(E, Hd, generator=g).cuda() * 0.1
    img, sc, layer, cw = _weight(qf, q), s.cuda(), _on(qf, up, down), [w.cuda() for w in wts]

    def step(x, r):
        y, h = qf.block_norm_rows(x, r, cw[0], cw[1])
        o = qf.fp8_linear(h, img, sc)
        y2, h2 = qf.block_norm_rows(o, y, cw[2], cw[3], alpha=0.5)
        logits = h2.float() @ router.t()
        m = qf.moe_few_tokens(h2, logits, *layer, k) if T <= 16 else qf.fp8_linear(h2, img, sc)
        y3, h3 = qf.block_norm_rows(m, y2, None, cw[0])
        return y, h, o, y2, h2, logits, m, y3, h3

    x, r = x0.cuda(), r0.cuda()
    want = step(x, r)
    torch.cuda.synchronize()
    ref, bound = H.product(want[1].cpu(), q, s, None, T > 16)
    H.within(want[2], ref, bound, H.BF16)
    if T <= 16:
        ref, bound = _reference(want[4].cpu(), want[5].cpu(), up, down, k, True)
        H.within(want[6], ref, bound, H.BF16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(x, r)  # the library product's workspaces exist before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step(x, r)
    for _ in range(3):
        graph.replay()
        again = step(x, r)
        torch.cuda.synchronize()
        for a, b, c in zip(got, want, again):
            assert torch.equal(a, b) and torch.equal(c, b)


def _weight(qf, q):
    return qf.fp8_to_tiled(q.cuda().t())
