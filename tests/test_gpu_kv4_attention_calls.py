"""Prompt chunks over the 4-bit cache as a program may call them: captured, on two streams at once, into the query itself, of
expanded queries, with one table row for several requests; against 64 bits and against the plain call."""
import pytest
import torch

from test_gpu_kv4_attention import _batch, _call, _check
import qwen_fastpath as qf

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32

# (requests' lengths, their new tokens, heads, kv heads, D): row tiles that fill the machine and that do not, single tokens beside
# chunks, single tokens alone with and without a split
BATCHES = [([900], [300], 16, 2, 128), ([560], [520], 64, 8, 64), ([500, 33, 1200, 7, 0, 64, 900], [150, 1, 0, 20, 12, 64, 1], 6, 1, 256),
           ([500, 33, 1200, 7, 0, 64, 900], [150, 1, 0, 20, 12, 64, 1], 16, 2, 128), ([3000], [3], 8, 2, 128), ([70, 9], [1, 1], 8, 2, 64)]


@pytest.mark.parametrize("i", range(len(BATCHES)))
def test_into_the_query_itself(i):
    s = _batch(i, BATCHES[i][0], BATCHES[i][1], *BATCHES[i][2:], 16)
    want = _call(s)
    _check(s, want)
    for _ in range(3):
        query = s["query"].cuda()
        how = dict(cu_q=s["cu"].int().cuda(), max_q=max(s["q"])) if len(set(s["q"])) > 1 else dict(q_len=s["q"][0])
        got = qf.kv4_attention(query, s["cache"], torch.tensor(s["seq"], dtype=I32).cuda(), s["table"].cuda(), s["scale"], out=query, **how)
        assert got is query and torch.equal(query, want)


@pytest.mark.parametrize("D,heads,kv", [(64, 4, 1), (128, 16, 2), (256, 6, 1)])
def test_a_captured_ragged_call(D, heads, kv):
    """Lengths and token counts that change under the graph, from all single tokens to one chunk, with eager calls and other
    tensors' frees between the replays; rows behind the last request's stay."""
    T, most = 260, 200
    plans = [([300, 40, 900, 5], [100, 1, 150, 5]), ([50, 60, 70, 80], [1, 1, 1, 1]), ([200, 0, 10, 999], [200, 0, 10, 1]),
             ([2, 700, 33, 64], [60, 0, 33, 64]), ([0, 0, 0, 0], [0, 0, 0, 0]), ([300, 40, 900, 5], [100, 1, 150, 5])]
    full = _batch(D, [999, 700, 900, 999], [65] * 4, heads, kv, D, 16)
    query = full["query"].cuda()
    seq, cu = torch.zeros(4, dtype=I32).cuda(), torch.zeros(5, dtype=I32).cuda()
    table, out = full["table"].cuda(), torch.full_like(query, 3.0)

    def call(to):
        return qf.kv4_attention(query, full["cache"], seq, table, full["scale"], cu_q=cu, max_q=most, out=to)
    call(out)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(out)
    for lengths, q in plans:
        cu.copy_(torch.tensor([0] + q).cumsum(0))
        seq.copy_(torch.tensor(lengths))
        out.fill_(3.0)
        graph.replay()
        eager = call(torch.full_like(out, 3.0))
        torch.randn(1 << 20, device="cuda").sum().item()
        first = out.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(first, eager)
        used = sum(q)
        assert bool((out[used:] == 3.0).all())
        s = {**full, "query": full["query"][:used], "q": q, "seq": lengths, "cu": torch.tensor([0] + q).cumsum(0)}
        _check(s, out[:used])


def test_chunks_on_two_streams():
    batches = [_batch(20 + i, *BATCHES[i][:2], *BATCHES[i][2:], 16) for i in (0, 1, 3)]
    want = [_call(s) for s in batches]
    args = [(s["query"].cuda(), s["cache"], torch.tensor(s["seq"], dtype=I32).cuda(), s["table"].cuda(), s["scale"]) for s in batches]
    how = [dict(cu_q=s["cu"].int().cuda(), max_q=max(s["q"])) for s in batches]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in batches], [[] for _ in batches]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(qf.kv4_attention(*args[i], **how[i]))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert all(torch.equal(w, x) for x in got[i])


@pytest.mark.parametrize("q", [2, 90])
def test_one_query_for_all_tokens_and_one_row_for_all_requests(q):
    s = _batch(31, [200], [q], 8, 2, 128, 16)
    one = s["query"][:1]
    s.update(query=one.expand(3 * q, 8, 128), seq=[200, 150, 77], q=[q] * 3, cu=torch.arange(4) * q, keys=s["keys"] * 3, vals=s["vals"] * 3)
    row = s["table"].cuda()
    got = qf.kv4_attention(one.cuda().expand(3 * q, 8, 128), s["cache"], torch.tensor(s["seq"], dtype=I32).cuda(),
                           row.expand(3, row.shape[1]), s["scale"], q_len=q)
    _check(s, got)


def test_the_fewest_and_the_most_heads():
    """A head of its own for each kv head, one head in all, and 64 heads over one, of a chunk and of single tokens."""
    for heads, kv in ((1, 1), (16, 16), (64, 1)):
        for q in (1, 70):
            s = _batch(heads + q, [130], [q], heads, kv, 64, 16)
            _check(s, _call(s))
    s = _batch(1, [40], [1], 96, 1, 64, 16)  # more heads over one than the split kernel's rows: a token alone takes a row tile
    _check(s, _call(s))
    s = _batch(2, [40, 9, 30], [1, 0, 5], 96, 1, 128, 16)
    _check(s, _call(s))
