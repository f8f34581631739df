"""Block-scaled FP8 products on the GPU against 64-bit references (block_helpers) with derived bounds: both arithmetics,
both weight layouts, odd sizes, and the calls the documentation allows."""
import pytest
import torch

import block_helpers as H

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def qf():
    import qwen_fastpath
    return qwen_fastpath


def _weight_on(qf, q, tiled):
    return qf.fp8_to_tiled(q.cuda().t()) if tiled else q.cuda().t()


def _check(qf, M, N, K, tiled, bias, out, a8, seed=0):
    g = H.gen(seed)
    q, s = H.weight(g, N, K)
    x = H.rows(g, M, K)
    b = torch.randn(N, generator=g).to(BF16) if bias else None
    mm = qf.fp8_w8a8_mm if a8 else qf.fp8_w8a16_mm
    y = mm(x.cuda(), _weight_on(qf, q, tiled), s.cuda(), out, None if b is None else b.cuda(), out_features=N)
    torch.cuda.synchronize()
    assert y.dtype == out
    ref, bound = H.product(x, q, s, b, a8)
    H.within(y, ref, bound, H.BF16 if out == BF16 else H.F32)
    return y


@pytest.mark.parametrize("N,K", [(64, 128), (7, 64), (1, 192), (2500, 1088), (130, 640)])
def test_tiled_image(qf, N, K):
    q, _ = H.weight(H.gen(N), N, K)
    image = qf.fp8_to_tiled(q.cuda().t())
    assert torch.equal(image.cpu().view(torch.uint8), H.tiles(q).view(torch.uint8))
    assert torch.equal(qf.fp8_from_tiled(image, N, K).cpu().view(torch.uint8), q.t().view(torch.uint8))


@pytest.mark.parametrize("tiled", [True, False])
@pytest.mark.parametrize("M,N,K", [(1, 16, 64), (1, 128, 128), (3, 1, 64), (16, 17, 192), (5, 300, 1088), (16, 2500, 2112),
                                   (2, 129, 8192), (9, 640, 17408), (7, 16640, 256), (16, 33000, 320)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_decode(qf, M, N, K, tiled, out):
    _check(qf, M, N, K, tiled, M % 2 == 1, out, False, seed=M + N)


# each form of the kernel (blocks a wavefront, x in LDS for up to 4, 8 and 16 tokens or in registers) with and without K splits
@pytest.mark.parametrize("tiled", [True, False])
@pytest.mark.parametrize("M,N,K", [
    (15, 16672, 1920), (15, 4144, 7680), (4, 16, 5248), (8, 16, 3968), (15, 16, 2560), (9, 1376, 3968), (9, 8352, 3968),
    (9, 16, 46336), (1, 16, 2176), (1, 16, 18688), (5, 16, 2176), (5, 16, 18688), (9, 16, 2176), (9, 16, 21248), (9, 2112, 4736),
    (9, 16, 50304), (1, 16, 4224), (1, 16, 50304), (5, 16, 4224), (5, 288, 50304), (9, 4144, 2944), (9, 608, 25088), (5, 2736, 6528),
    (9, 480, 50304), (1, 16, 6272), (1, 1040, 18688), (5, 1376, 6272), (5, 416, 50304), (9, 16, 3200), (9, 16, 34944),
    (9, 4144, 3968), (12, 16, 15104), (9, 1040, 27264), (9, 21328, 2048)])
def test_decode_forms(qf, M, N, K, tiled):
    g = H.gen(K)
    q, s = H.weight(g, N, K)
    x, bias = H.rows(g, M, K), torch.randn(N, generator=g).to(BF16)
    y = qf.fp8_w8a16_mm(x.cuda(), _weight_on(qf, q, tiled), s.cuda(), F32, bias.cuda(), N).cpu()
    for b in {0, (N - 1) // 256, (N - 1) // 128}:  # channels of these blocks
        at = slice(128 * b, min(128 * b + 128, N))
        ref, bound = H.product(x, q[at], s[b:b + 1], bias[at], False)
        H.within(y[:, at], ref, bound, H.F32)


@pytest.mark.parametrize("M", range(1, 17))
def test_decode_every_width(qf, M):
    _check(qf, M, 272, 640, M % 2 == 0, False, BF16, False, seed=M)


@pytest.mark.parametrize("M,K", [(1, 64), (3, 192), (16, 128), (17, 1088), (333, 5120), (2, 17408)])
def test_quantiser_bits(qf, M, K):
    x = H.rows(H.gen(M), M, K)
    x[0, :64] = 0
    x[M - 1, K - 64:] = 0
    x[M // 2, 0] = 3e38
    q, s = qf.quantize_tokens_fp8(x.cuda())
    qr, sr = H.quantize(x)
    assert torch.equal(s.cpu(), sr)
    assert torch.equal(q.cpu().view(torch.uint8) , qr.view(torch.uint8))


def test_quantiser_rounds_as_the_division(qf):
    """Every sign, exponent and significand against maxima of all kinds: bit for bit, signed zeros among them."""
    g = H.gen(9)
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    x = x[x.isfinite()][:65024].view(508, 128).clone()       # blocks of like magnitude
    y = x.flatten()[torch.randperm(65024, generator=g)].view(508, 128)  # and of unlike
    z = (H.rows(g, 508, 128).float() * 2.0 ** torch.randint(-126, 100, (508, 1), generator=g)).to(BF16)
    x = torch.cat([x, y, z], 1)
    q, s = qf.quantize_tokens_fp8(x.cuda())
    qr, sr = H.quantize(x)
    assert torch.equal(s.cpu(), sr)
    assert torch.equal(q.cpu().view(torch.uint8), qr.view(torch.uint8))


def test_quantiser_tiny_and_not_finite(qf):
    x = torch.zeros(4, 256)
    x[0, :8] = torch.tensor([1, -2, 3, -4, 5, 100, 333, 127.]) * 2.0 ** -133  # subnormal in bf16
    x[1, 5] = float("inf")
    x[2, 200] = float("nan")
    x[3, 7] = 2.0 ** -126
    x = x.to(BF16)
    q, s = qf.quantize_tokens_fp8(x.cuda())
    qr, sr = H.quantize(x)
    v = q.cpu().double() * s.cpu().double().repeat_interleave(128, 1)
    r = qr.double() * sr.double().repeat_interleave(128, 1)
    assert torch.equal(torch.isnan(v[1, :128]), torch.isnan(r[1, :128])) and v[1, 128:].eq(0).all()
    assert torch.isnan(v[2]).any() and v[2, :128].eq(0).all()
    for m in (0, 3):
        assert torch.equal(q.cpu().view(torch.uint8)[m], qr.view(torch.uint8)[m]) and torch.equal(s.cpu()[m], sr[m])


@pytest.mark.parametrize("tiled", [True, False])
@pytest.mark.parametrize("M,N,K", [(1, 16, 64), (17, 1, 128), (17, 128, 192), (64, 300, 1088), (77, 2500, 2112),
                                   (129, 5120, 256), (300, 130, 8256), (200, 26000, 192), (1030, 8200, 320), (513, 127, 64)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_w8a8(qf, M, N, K, tiled, out):
    _check(qf, M, N, K, tiled, M % 2 == 1, out, True, seed=M + N)


# a whole round of the largest tiles, tokens that end inside one; whole rounds and a second launch for the channels behind
# (of each smaller tile); each tile with K splits
@pytest.mark.parametrize("tiled", [True, False])
@pytest.mark.parametrize("M,N,K", [
    (1000, 16384, 320), (260, 33000, 2624), (2917, 11832, 512), (2917, 5834, 768), (2751, 6068, 640), (2309, 2096, 7424),
    (2178, 1862, 4864), (1286, 912, 4864), (852, 1157, 4224), (904, 663, 11648), (904, 663, 5632), (598, 777, 3456), (532, 588, 9600)])
def test_w8a8_wide(qf, M, N, K, tiled):
    g = H.gen(N)
    q, s = H.weight(g, N, K)
    x, bias = H.rows(g, M, K), torch.randn(N, generator=g).to(BF16)
    w = qf.fp8_to_tiled(q.cuda().t()) if tiled else q.cuda().t()
    y = qf.fp8_w8a8_mm(x.cuda(), w, s.cuda(), bias=bias.cuda(), out_features=N).cpu()
    rows = torch.tensor([0, 255, 256, M // 2, M - 1])
    for b in {min(b, (N - 1) // 128) for b in (0, N // 256, 31, 255, N // 128 - 1, N // 128)}:  # channels of these blocks
        at = slice(128 * b, min(128 * b + 128, N))
        ref, bound = H.product(x[rows], q[at], s[b:b + 1], bias[at], True)
        H.within(y[rows][:, at], ref, bound, H.BF16)


def test_linear_picks_by_rows_and_keeps_leading_dims(qf):
    g = H.gen(5)
    q, s = H.weight(g, 200, 256)
    x = H.rows(g, 24, 256).cuda()
    w, s = q.cuda().t(), s.cuda()
    assert torch.equal(qf.fp8_linear(x[:16], w, s), qf.fp8_w8a16_mm(x[:16], w, s))
    assert torch.equal(qf.fp8_linear(x, w, s), qf.fp8_w8a8_mm(x, w, s))
    assert torch.equal(qf.fp8_linear(x.view(2, 3, 4, 256), w, s), qf.fp8_linear(x, w, s).view(2, 3, 4, 200))
    assert torch.equal(torch.ops.qwen_fastpath.qf_fp8_linear(x, w, s), qf.fp8_linear(x, w, s))
    assert qf.fp8_linear(x[:0], w, s).shape == (0, 200)
    assert qf.fp8_linear(x[:0].view(2, 0, 256), w, s).shape == (2, 0, 200)
    assert torch.equal(qf.fp8_linear(x[0], w, s), qf.fp8_linear(x[:1], w, s)[0])


@pytest.mark.parametrize("M,N,K", [(1, 200, 256), (16, 64, 8192), (40, 130, 320)])
def test_plain_calls_agree_with_the_long_way(qf, monkeypatch, M, N, K):
    import qwen_fastpath._qf_block_call as plain
    g = H.gen(M)
    q, s = H.weight(g, N, K)
    x, w, s, bias = H.rows(g, M, K).cuda(), q.cuda().t(), s.cuda(), torch.randn(N, generator=g).to(BF16).cuda()
    image = qf.fp8_to_tiled(w)
    calls = [lambda: qf.fp8_linear(x, w, s), lambda: qf.fp8_linear(x, image, s, bias, N), lambda: qf.fp8_w8a8_mm(x, w, s, F32),
             lambda: qf.fp8_w8a8_mm(x, image, s, bias=bias, out_features=N)]
    took = []
    real = plain.product
    monkeypatch.setattr(plain, "product", lambda *a: took.append(real(*a)) or took[-1])
    short = [f() for f in calls]
    assert len(took) == len(calls) and all(t is not None for t in took)
    monkeypatch.setattr(plain, "product", lambda *a: None)
    for a, f in zip(short, calls):
        b = f()
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_wrong_calls_on_the_gpu(qf):
    g = H.gen(0)
    q, s = H.weight(g, 200, 256)
    x, w, s = H.rows(g, 24, 256).cuda(), q.cuda().t(), s.cuda()
    image, bias = qf.fp8_to_tiled(w), torch.zeros(200, dtype=BF16, device="cuda")
    for f in (lambda: qf.fp8_w8a8_mm(x, w, s, torch.float16), lambda: qf.fp8_linear(x.half(), w, s), lambda: qf.fp8_linear(x, w, s.half()),
              lambda: qf.fp8_linear(x, w.view(torch.uint8), s), lambda: qf.fp8_linear(x, w, s, bias.float()),
              lambda: qf.fp8_linear(x, w, s, bias[:199])):
        with pytest.raises(TypeError):
            f()
    for f in (lambda: qf.fp8_linear(x, image, s, None, -1), lambda: qf.fp8_linear(x, image, s, None, 0), lambda: qf.fp8_linear(x, image, s, None, 192),
              lambda: qf.fp8_linear(x, w, s, None, 199), lambda: qf.fp8_linear(x, w, s[:, :1]), lambda: qf.fp8_linear(x[:, :192], w, s),
              lambda: qf.fp8_linear(x, w, s.cpu()), lambda: qf.fp8_linear(x, w.cpu(), s), lambda: qf.fp8_w8a16_mm(x, w, s),
              lambda: qf.fp8_linear(x[:, :100].contiguous(), w[:100], s)):
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("M", [5, 40, 300])
def test_strided_and_unaligned_inputs(qf, M):
    g = H.gen(M)
    q, s = H.weight(g, 200, 320)
    x = H.rows(g, M, 320)
    w, sc = q.cuda().t(), s.cuda()
    y = qf.fp8_linear(x.cuda(), w, sc)
    wide = torch.zeros(M, 400, dtype=BF16, device="cuda")
    wide[:, 8:328] = x.cuda()
    assert torch.equal(qf.fp8_linear(wide[:, 8:328], w, sc), y)
    wide[:, 3:323] = x.cuda()
    assert torch.equal(qf.fp8_linear(wide[:, 3:323], w, sc), y)
    assert torch.equal(qf.fp8_linear(x.cuda().t().contiguous().t(), w, sc), y)
    rows = torch.zeros(200, 352, dtype=torch.uint8, device="cuda")
    rows[:, 16:336] = q.cuda().view(torch.uint8)
    assert torch.equal(qf.fp8_linear(x.cuda(), rows[:, 16:336].view(H.FP8).t(), sc), y)


@pytest.mark.parametrize("M", [4, 40])
def test_not_finite_values_stay_in_their_rows_and_channels(qf, M):
    g = H.gen(M)
    q, s = H.weight(g, 200, 320)
    x = H.rows(g, M, 320)
    x[1, 300] = float("nan")
    qb = q.view(torch.uint8)
    qb[70, 11] = 0x7f  # NaN
    y = qf.fp8_linear(x.cuda(), q.cuda().t(), s.cuda()).cpu()
    nan = torch.zeros(M, 200, dtype=torch.bool)
    nan[1] = True
    nan[:, 70] = True
    assert torch.equal(torch.isnan(y), nan)


@pytest.mark.parametrize("M,N,K", [(5, 2500, 1088), (9, 16, 18688), (16, 2560, 4352), (77, 2500, 2112), (300, 512, 1024), (852, 1157, 4224)])
def test_graph_replays_and_repeats_bitwise(qf, M, N, K):
    g = H.gen(M)
    q, s = H.weight(g, N, K)
    w, s = _weight_on(qf, q, True), s.cuda()
    x = H.rows(g, M, K).cuda()
    other = H.rows(g, M, K).cuda()
    want, want_other = (qf.fp8_linear(v, w, s, out_features=N) for v in (x, other))
    static = x.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = qf.fp8_linear(static, w, s, out_features=N)
        z = qf.fp8_linear(static, w, s, out_features=N)
    for v, ref in ((x, want), (other, want_other), (x, want)):
        static.copy_(v)
        graph.replay()
        assert torch.equal(qf.fp8_linear(v, w, s, out_features=N), ref)  # the program's own work between replays
        torch.cuda.synchronize()
        assert torch.equal(y, ref) and torch.equal(z, ref)


@pytest.mark.parametrize("M", [16, 60])
def test_two_graphs_at_once(qf, M):
    """Graphs captured on one stream, their K splits' workspaces their own: replayed on two streams, eager calls beside."""
    g = H.gen(M)
    q, s = H.weight(g, 1200, 4352)
    w, s = _weight_on(qf, q, True), s.cuda()
    xs = [H.rows(g, M, 4352).cuda() for _ in range(3)]
    want = [qf.fp8_linear(x, w, s, out_features=1200) for x in xs]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for x in xs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(qf.fp8_linear(x, w, s, out_features=1200))
        graphs.append(graph)
    sides = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        for side, graph in zip(sides, graphs):
            with torch.cuda.stream(side):
                graph.replay()
        eager = qf.fp8_linear(xs[2], w, s, out_features=1200)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])


def test_calls_on_two_streams_at_once(qf):
    g = H.gen(9)
    q, s = H.weight(g, 1000, 2112)
    w, s = q.cuda().t(), s.cuda()
    xs = [H.rows(g, M, 2112).cuda() for M in (40, 300, 7, 129)]
    want = [qf.fp8_linear(x, w, s) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(qf.fp8_linear(xs[i // 2], w, s))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i // 2])
