"""A step's tables, entry by entry against the same steps in Python."""
import random

import pytest
import torch

import kv4_helpers as H
import qwen_fastpath as qf

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _state(seed, B, page, most_context, most_q, spare=4, idle=0.1, extra=0.2):
    r = random.Random(seed)
    context = [r.randint(0, most_context) for _ in range(B)]
    q = [0 if r.random() < idle else r.randint(1, most_q) for _ in range(B)]
    held = [-(-c // page) + (r.random() < extra) for c in context]
    width = max(max(h, -(-(c + n) // page)) for h, c, n in zip(held, context, q)) + 2
    need = sum(max(0, -(-(c + n) // page) - h) for h, c, n in zip(held, context, q))
    ids = list(range(sum(held) + need + spare))
    r.shuffle(ids)
    table = torch.full((B, width), -7, dtype=I32)
    for b, h in enumerate(held):
        table[b, :h] = torch.tensor([ids.pop() for _ in range(h)], dtype=I32)
    return dict(context=torch.tensor(context, dtype=I32), q=torch.tensor(q, dtype=I32), held=torch.tensor(held, dtype=I32), table=table,
                stack=torch.tensor(ids + [-1, -1], dtype=I32), count=len(ids), page=page, tokens=sum(q))


def _run(s, tokens=None, table=None):
    tokens = s["tokens"] if tokens is None else tokens
    want_table = s["table"].clone()
    want = H.tables(s["context"], s["q"], s["held"], want_table, s["stack"].tolist(), s["count"], s["page"], tokens)
    table = s["table"].cuda() if table is None else table
    got = qf.step_tables(s["context"].cuda(), s["q"].cuda(), s["held"].cuda(), table, s["stack"].cuda(),
                         torch.tensor([s["count"]], dtype=I32).cuda(), s["page"], tokens)
    for name, v in want.items():
        assert getattr(got, name).tolist() == v, name
    assert torch.equal(table.cpu(), want_table)
    return got


@pytest.mark.parametrize("B,page,context,q,pad", [
    (1, 16, 1000, 5, 0), (1, 16, 0, 1, 0), (1, 64, 100, 4000, 9), (2, 1, 30, 3, 1), (3, 16, 5, 300, 0), (63, 48, 900, 6, 2),
    (64, 16, 64, 1, 0), (65, 16, 64, 2, 100), (257, 33, 3000, 40, 0), (700, 16, 500, 8, 13), (4096, 16, 100, 3, 1),
    (4095, 128, 2000, 2, 0)])
def test_against_python(B, page, context, q, pad):
    s = _state(B + page, B, page, context, q)
    got = _run(s, s["tokens"] + pad)
    assert got.fits.item() == 1 and [t.dtype for t in got] == [I32, I32, torch.int64, torch.int64, I32, I32, I32]


def test_idle_requests_only():
    s = _state(1, 5, 16, 100, 1, idle=1.0)
    assert s["tokens"] == 0
    _run(s, 0)
    _run(s, 3)


@pytest.mark.parametrize("name,change", [
    ("tokens", lambda s: s.update(tokens=s["tokens"] - 1)), ("stack", lambda s: s.update(count=0)),
    ("count past the stack", lambda s: s.update(count=len(s["stack"]) + 1)), ("negative count", lambda s: s.update(count=-1)),
    ("context", lambda s: s["context"].__setitem__(2, -1)), ("query", lambda s: s["q"].__setitem__(3, -1)),
    ("held", lambda s: s["held"].__setitem__(1, -1)), ("held past the row", lambda s: s["held"].__setitem__(1, 1000)),
    ("pages past the row", lambda s: s["context"].__setitem__(4, 100000)),
    ("sum past 2^31", lambda s: (s["context"].__setitem__(0, 2 ** 31 - 1), s["q"].__setitem__(0, 5))),
    ("many tokens", lambda s: s["q"].fill_(2 ** 31 - 1))])
def test_a_step_that_does_not_fit_takes_nothing(name, change):
    s = _state(9, 7, 16, 300, 40, idle=0.0)
    change(s)
    got = _run(s)
    assert got.fits.item() == 0


def test_exactly_the_stack():
    s = _state(10, 30, 16, 200, 90, spare=0)
    assert _run(s).free_count.item() == 0


def test_strides_and_wider_tables():
    """A table with more rows than requests and a row stride; lengths that are views."""
    s = _state(11, 6, 16, 200, 30)
    wide = torch.full((9, s["table"].shape[1] + 5), 77, dtype=I32, device="cuda")
    wide[:6, :s["table"].shape[1]] = s["table"].cuda()
    _run(s, table=wide[:6, :s["table"].shape[1]])
    assert bool((wide[6:] == 77).all()) and bool((wide[:, s["table"].shape[1]:] == 77).all())
    got = qf.step_tables(torch.stack([s["context"]] * 2, 1).cuda()[:, 0], s["q"].cuda(), s["held"].cuda(), wide, s["stack"].cuda(),
                         torch.tensor([s["count"]], dtype=I32).cuda(), s["page"], s["tokens"])
    assert got.cu_q[-1].item() == s["tokens"]


def test_a_loop_on_the_gpu():
    """Steps one after the other from the returned tensors, without a word from the host; the pages of all requests stay apart."""
    B, page = 23, 16
    g = H.gen(4)
    stack = torch.randperm(1500, generator=g).int()
    context, held = torch.zeros(B, dtype=I32).cuda(), torch.zeros(B, dtype=I32).cuda()
    count = torch.tensor([1500], dtype=I32).cuda()
    table = torch.zeros(B, 120, dtype=I32).cuda()
    h_context, h_held, h_table, h_count = torch.zeros(B, dtype=I32), torch.zeros(B, dtype=I32), torch.zeros(B, 120, dtype=I32), 1500
    for step in range(12):
        q = torch.randint(0, 90 if step % 3 == 0 else 6, (B,), generator=g).int()
        t = qf.step_tables(context, q.cuda(), held, table, stack.cuda(), count, page, 2000)
        want = H.tables(h_context, q, h_held, h_table, stack.tolist(), h_count, page, 2000)
        for name, v in want.items():
            assert getattr(t, name).tolist() == v, (step, name)
        taken = torch.randint(0, 2, (B,), generator=g).int()  # some of the drafted tokens are rejected
        context, held, count = (t.seq_lens - torch.minimum(taken.cuda(), q.cuda())).int(), t.held, t.free_count
        h_context, h_held, h_count = context.cpu(), held.cpu(), int(count)
    used = torch.cat([h_table[b, :h_held[b]] for b in range(B)])
    assert len(used.unique()) == len(used) and torch.equal(table.cpu(), h_table)


def test_captured():
    s = _state(12, 40, 16, 500, 20)
    dev = {n: s[n].cuda() for n in ("context", "q", "held", "table", "stack")}
    count = torch.tensor([s["count"]], dtype=I32).cuda()
    call = lambda: qf.step_tables(dev["context"], dev["q"], dev["held"], dev["table"], dev["stack"], count, 16, 900)  # noqa: E731
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = call()
    for seed in (12, 13, 14):
        n = _state(seed, 40, 16, 500, 20)
        table = s["table"].clone()
        n["table"] = torch.full_like(table, -7)
        w = min(table.shape[1], _state(seed, 40, 16, 500, 20)["table"].shape[1])
        n["table"][:, :w] = _state(seed, 40, 16, 500, 20)["table"][:, :w]
        n["stack"] = torch.nn.functional.pad(n["stack"], (0, max(0, len(s["stack"]) - len(n["stack"]))))[:len(s["stack"])]
        n["count"] = min(n["count"], len(s["stack"]))
        for name in dev:
            dev[name].copy_(n[name])
        count.fill_(n["count"])
        want = H.tables(n["context"], n["q"], n["held"], n["table"], n["stack"].tolist(), n["count"], 16, 900)
        graph.replay()
        torch.cuda.synchronize()
        for name, v in want.items():
            assert getattr(t, name).tolist() == v, (seed, name)
        assert torch.equal(dev["table"].cpu(), n["table"])
