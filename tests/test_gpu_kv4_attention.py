"""Attention over the 4-bit cache against 64 bits of the values that the cache stands for (bounds in kv4_helpers)."""
import math

import pytest
import torch

import kv4_helpers as H
import qwen_fastpath as qf

pytestmark = pytest.mark.gpu
BF16, U8, I32 = torch.bfloat16, torch.uint8, torch.int32


def _batch(seed, seq, q, heads, kv, D, page, poison=True, spread=1.0):
    """Requests of these lengths and query tokens in a shuffled cache.  Whatever no request holds (other positions of the last
    pages, other pages) is NaN with `poison`."""
    g = H.gen(seed)
    blocks, table = H.paged(g, seq, page)
    keys, vals = [], []
    cache = torch.full((blocks, kv, page // 16, 17 * D), 255 if poison else 0, dtype=U8).cuda()
    for b, n in enumerate(seq):
        k = torch.randn(n, kv, D, generator=g) * spread
        k[..., 3::31] *= 5
        v = torch.randn(n, kv, D, generator=g) * torch.exp(torch.randn(n, kv, 1, generator=g))
        k, v = k.to(BF16), v.to(BF16)
        if n:
            qf.kv4_store(k.cuda(), v.cuda(), cache, H.slots_of(table, b, n, page).cuda())
        keys.append(H.rounded(k) if n else k.double())
        vals.append(H.rounded(v) if n else v.double())
    cu = torch.tensor([0] + q).cumsum(0)
    query = torch.randn(int(cu[-1]), heads, D, generator=g).to(BF16)
    return dict(query=query, cache=cache, seq=seq, q=q, cu=cu, table=table, keys=keys, vals=vals, scale=D ** -0.5)


def _call(s, ragged=None, **kw):
    ragged = len(set(s["q"])) > 1 if ragged is None else ragged
    how = dict(cu_q=s["cu"].int().cuda(), max_q=max(s["q"])) if ragged else dict(q_len=s["q"][0])
    return qf.kv4_attention(s["query"].cuda(), s["cache"], torch.tensor(s["seq"], dtype=I32).cuda(), s["table"].cuda(), s["scale"],
                            **{**how, **kw})


def _check(s, got):
    want, slack = H.attention(s["query"], s["keys"], s["vals"], s["cu"], s["seq"], s["scale"])
    H.near(got, want, slack)
    empty = torch.cat([torch.arange(n) < n - L for n, L in zip(s["q"], s["seq"])])
    assert not got.cpu()[empty].any()


# ---- decode and verification ----

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("seq,q,heads,kv,page", [
    ([1], 1, 1, 1, 16), ([16], 1, 2, 1, 16), ([17], 1, 8, 1, 16), ([31], 2, 3, 3, 16), ([33], 3, 4, 2, 32), ([127], 1, 8, 8, 16),
    ([129], 1, 16, 1, 48), ([300], 5, 6, 2, 16), ([1000], 1, 8, 1, 64), ([2000], 3, 12, 2, 16), ([4100], 4, 16, 1, 16),
    ([700, 3, 0, 1300], 1, 4, 2, 16), ([64, 65, 63, 1, 2], 4, 8, 2, 16), ([5, 900, 31, 32, 33, 2], 5, 24, 2, 48)])
def test_uniform(D, seq, q, heads, kv, page):
    s = _batch(len(seq) + D + q, seq, [q] * len(seq), heads, kv, D, page)
    _check(s, _call(s))


@pytest.mark.parametrize("rows", range(1, 9))
@pytest.mark.parametrize("q", [1, 2, 4, 8])
def test_every_count_of_rows(rows, q):
    """Packed rows of 1 to 64: every row tile and its last rows."""
    s = _batch(rows * q, [260, 41], [q] * 2, rows * 2, 2, 128, 16)
    _check(s, _call(s))


@pytest.mark.parametrize("D,heads,kv", [(64, 8, 1), (128, 6, 3), (256, 6, 1)])
def test_ragged_few_tokens(D, heads, kv):
    s = _batch(D, [50, 0, 700, 9, 333, 2, 17], [3, 0, 1, 8, 0, 5, 2], heads, kv, D, 16)
    _check(s, _call(s))


def test_many_requests():
    """More requests than lanes of a wavefront, than compute units, some without tokens or positions."""
    g = H.gen(0)
    seq = [int(torch.randint(0, 90, (1,), generator=g)) for _ in range(300)]
    q = [int(torch.randint(0, 4, (1,), generator=g)) for _ in range(300)]
    s = _batch(1, seq, q, 4, 2, 64, 16)
    _check(s, _call(s))
    s = _batch(2, [9000] + [20] * 129, [1] * 130, 4, 4, 64, 64)
    _check(s, _call(s))


def test_long_context():
    s = _batch(3, [38000], [2], 12, 2, 256, 16)
    _check(s, _call(s))


# ---- prompt chunks ----

@pytest.mark.parametrize("D,seq,q,heads,kv,page", [
    (64, [65], 65, 2, 1, 16), (128, [200], 200, 4, 4, 16), (256, [90], 70, 6, 2, 16), (128, [1000], 129, 8, 1, 64), (64, [700], 300, 5, 1, 48),
    (256, [513], 257, 2, 2, 32), (128, [33], 100, 8, 1, 16), (128, [3000], 40, 16, 2, 16), (128, [600], 600, 8, 2, 16)])
def test_chunk(D, seq, q, heads, kv, page):
    s = _batch(D + q, seq, [q], heads, kv, D, page)
    _check(s, _call(s))


@pytest.mark.parametrize("D,heads,kv", [(64, 4, 2), (128, 16, 2), (256, 6, 1)])
def test_ragged_chunks(D, heads, kv):
    """Chunks beside single tokens, requests without tokens, without positions, and shorter than their queries."""
    s = _batch(D, [500, 33, 1200, 7, 0, 64, 900], [150, 1, 0, 20, 12, 64, 1], heads, kv, D, 16)
    _check(s, _call(s))


# ---- masks, infinities, what must not be touched ----

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q,n", [(3, 200), (90, 200), (90, 1500)])
def test_nan_behind_a_query_stays_there(D, q, n):
    """A key or a value that is NaN changes the queries that see it, and no earlier one."""
    s = _batch(D + q, [n], [q], 4, 2, D, 16)
    for pos, where in ((n - 1, "vals"), (n - 2, "keys"), (n - q, "vals")):
        k, v = s["keys"][0][pos:pos + 1].clone().to(BF16), s["vals"][0][pos:pos + 1].clone().to(BF16)
        (k if where == "keys" else v)[0, 1, 5] = float("inf")
        cache = s["cache"].clone()
        qf.kv4_store(k.cuda(), v.cuda(), cache, H.slots_of(s["table"], 0, n, 16)[pos:pos + 1].cuda())
        bad = {**s, "cache": cache, "keys": [s["keys"][0].clone()], "vals": [s["vals"][0].clone()]}
        bad[where][0][pos, 1, :32] = math.nan
        got = _call(bad).cpu()
        want, slack = H.attention(s["query"], s["keys"], s["vals"], s["cu"], s["seq"], s["scale"])
        sees = n - q + torch.arange(q) >= pos
        for h in range(4):
            if h // 2 == 0:
                H.near(got[:, h], want[:, h], slack[:, h])
                continue
            H.near(got[~sees, h], want[~sees, h], slack[~sees, h])
            part = slice(0, 32) if where == "vals" else slice(0, D)
            assert got[sees, h, part].isnan().all()
            if where == "vals":
                H.near(got[sees, h, 32:], want[sees, h, 32:], slack[sees, h, 32:])


def test_queries_with_infinities():
    s = _batch(7, [100], [3], 4, 2, 128, 16)
    s["query"][1, 2, 7] = float("nan")
    got = _call(s)
    want, slack = H.attention(s["query"], s["keys"], s["vals"], s["cu"], s["seq"], s["scale"])
    assert got[1, 2].isnan().all()
    keep = torch.ones(3, 4, dtype=torch.bool)
    keep[1, 2] = False
    H.near(got.cpu()[keep], want[keep], slack[keep])


@pytest.mark.parametrize("scale", [0.0, -0.09, 3.0])
def test_scales(scale):
    s = _batch(8, [333], [2], 4, 1, 128, 16, spread=2.0)
    s["scale"] = scale
    _check(s, _call(s))
    s = _batch(8, [333], [70], 4, 1, 128, 16, spread=2.0)
    s["scale"] = scale
    _check(s, _call(s))


@pytest.mark.parametrize("q", [[2, 0, 3], [40, 0, 90]])
def test_rows_behind_the_last_sequence_stay(q):
    s = _batch(9, [100, 30, 95], q, 8, 2, 128, 16)
    T = sum(q)
    query = torch.randn(T + 5, 8, 128, generator=H.gen(1)).to(BF16)
    query[:T] = s["query"]
    out = torch.full((T + 5, 8, 128), 3.0, dtype=BF16, device="cuda")
    got = _call({**s, "query": query}, ragged=True, out=out)
    assert got is out and bool((out[T:] == 3.0).all())
    _check(s, out[:T])
    uniform = _batch(10, [100, 30], [2, 2], 8, 2, 128, 16)
    query[:4] = uniform["query"]
    out.fill_(3.0)
    _call({**uniform, "query": query}, out=out)
    assert bool((out[4:] == 3.0).all())
    _check(uniform, out[:4])


def test_lengths_and_ids_are_kept_inside():
    """Lengths past the table, negative ones, ids outside the cache, token counts past the query: nothing outside is read or
    written, and the other requests keep their results."""
    s = _batch(11, [40, 60, 50], [2, 2, 2], 4, 2, 64, 16, poison=False)
    want = _call(s)
    args = (s["query"].cuda(), s["cache"])
    table = s["table"].clone()
    for seq in ([40, 2 ** 31 - 1, 50], [40, -5, 50]):
        got = qf.kv4_attention(*args, torch.tensor(seq, dtype=I32).cuda(), table.cuda(), s["scale"], q_len=2)
        assert torch.equal(got[:2], want[:2]) and torch.equal(got[4:], want[4:])
    table[1] = torch.tensor([-1, 2 ** 31 - 1, len(s["cache"]), 5])[:table.shape[1]]
    got = qf.kv4_attention(*args, torch.tensor(s["seq"], dtype=I32).cuda(), table.cuda(), s["scale"], q_len=2)
    assert torch.equal(got[:2], want[:2]) and torch.equal(got[4:], want[4:])
    for cu in ([0, 2, 400, 500], [0, 2, -7, 6], [0, 2, 2 ** 31 - 1, -2 ** 31]):
        for most in (2, 70):
            out = torch.zeros(6, 4, 64, dtype=BF16, device="cuda")
            qf.kv4_attention(*args, torch.tensor(s["seq"], dtype=I32).cuda(), s["table"].cuda(), s["scale"],
                             cu_q=torch.tensor(cu, dtype=I32).cuda(), max_q=most, out=out)
            assert bool(out[:2].isfinite().all())


# ---- addresses ----

def test_strides_of_queries_outputs_tables_and_blocks():
    s = _batch(12, [300, 20], [3, 3], 4, 2, 128, 32)
    want = _call(s)
    wide = torch.zeros(6, 4, 2, 128, dtype=BF16, device="cuda")  # queries beside their gates
    wide[:, :, 0] = s["query"].cuda()
    layers = torch.zeros(s["cache"].shape[0], 3, *s["cache"].shape[1:], dtype=U8, device="cuda")
    layers[:, 1] = s["cache"]
    table = torch.zeros(5, s["table"].shape[1] + 3, dtype=I32, device="cuda")
    table[:2, :s["table"].shape[1]] = s["table"].cuda()
    seq = torch.tensor(s["seq"], dtype=I32).cuda()
    out = torch.zeros(6, 6, 136, dtype=BF16, device="cuda")
    got = qf.kv4_attention(wide[:, :, 0], layers[:, 1], seq, table, s["scale"], q_len=3, out=out[:, 1:5, :128])
    assert torch.equal(got, want) and not out[:, 0].any() and not out[:, 5].any() and not out[..., 128:].any()
    odd = torch.zeros(6, 4, 129, dtype=BF16, device="cuda")
    odd[..., 1:] = s["query"].cuda()
    got = qf.kv4_attention(odd[..., 1:], s["cache"], torch.stack([seq, seq], 1)[:, 0], s["table"].t().contiguous().t().cuda(), s["scale"],
                           q_len=3)
    assert torch.equal(got, want)


def test_offsets_past_32_bits():
    """Blocks that stand past 2^32 bytes."""
    D, page, kv = 256, 64, 4
    record = 17 * D * 4 * kv
    blocks = 2 ** 32 // record + 30
    cache = torch.empty(blocks, kv, 4, 17 * D, dtype=U8, device="cuda")
    s = _batch(13, [400], [2], 8, kv, D, page)
    order = torch.tensor([blocks - 1, 3, blocks - 9, blocks // 2, blocks - 4, 0, blocks - 2], dtype=I32)
    assert len(order) == s["table"].shape[1]
    cache[order.long().cuda()] = s["cache"][s["table"][0].long().cuda()]
    got = qf.kv4_attention(s["query"].cuda(), cache, torch.tensor([400], dtype=I32).cuda(), order[None].cuda(), s["scale"], q_len=2)
    assert torch.equal(got, _call(s))
    many = _batch(13, [400], [80], 8, kv, D, page)
    cache[order.long().cuda()] = many["cache"][many["table"][0].long().cuda()]
    got = qf.kv4_attention(many["query"].cuda(), cache, torch.tensor([400], dtype=I32).cuda(), order[None].cuda(), s["scale"], q_len=80)
    assert torch.equal(got, _call(many))


# ---- calls ----

def test_the_same_bits_every_time():
    for q in (2, 100):
        s = _batch(14, [3000, 200, 777], [q] * 3, 8, 2, 128, 16)
        first = _call(s)
        assert all(torch.equal(first, _call(s)) for _ in range(5))


def test_two_streams():
    a = _batch(15, [2000, 60], [2, 2], 8, 2, 128, 16)
    b = _batch(16, [1500, 900, 10], [1, 1, 1], 8, 2, 128, 16)
    want = _call(a), _call(b)
    torch.cuda.synchronize()
    args = [(s["query"].cuda(), s["cache"], torch.tensor(s["seq"], dtype=I32).cuda(), s["table"].cuda(), s["scale"]) for s in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, (st, q) in enumerate(zip(streams, (2, 1))):
            with torch.cuda.stream(st):
                got[i].append(qf.kv4_attention(*args[i], q_len=q))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(want[i], x) for x in got[i])


def test_two_graphs_replayed_in_turn():
    """Each graph with its own workspace, eager calls between the replays, lengths that change under the graph."""
    a = _batch(17, [2500], [3], 8, 2, 128, 16)
    b = _batch(18, [300, 1700, 40], [1, 1, 1], 16, 4, 64, 16)
    sets = []
    for s in (a, b):
        t = dict(query=s["query"].cuda(), cache=s["cache"], seq=torch.tensor(s["seq"], dtype=I32).cuda(), table=s["table"].cuda())
        call = lambda t=t, s=s: qf.kv4_attention(t["query"], t["cache"], t["seq"], t["table"], s["scale"], q_len=s["q"][0])  # noqa: E731
        call()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = call()
        sets.append((s, t, graph, out))
    for cut in (0, 700, 5, 1200, 0):
        for s, t, graph, out in sets:
            seq = [max(s["q"][0], n - cut) for n in s["seq"]]
            t["seq"].copy_(torch.tensor(seq, dtype=I32))
            graph.replay()
            eager = qf.kv4_attention(t["query"], t["cache"], t["seq"], t["table"], s["scale"], q_len=s["q"][0])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
            _check({**s, "seq": seq}, out)
