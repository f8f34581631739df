"""The operators as a serving loop runs them: the step's tables, then for each layer the norms with rotation and the write, and
the attention; against the same steps in 64 bits, eager and as one captured step."""
import pytest
import torch

import kv4_helpers as H
import qwen_fastpath as qf
from qwen_fastpath import spec_attn

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
B, HEADS, KV, D, PAGE, LAYERS, ROT = 5, 6, 2, 128, 16, 2, 64


class Loop:
    """What stands on the GPU between steps."""

    def __init__(self, seed):
        g = H.gen(seed)
        self.context, self.held = torch.zeros(B, dtype=I32).cuda(), torch.zeros(B, dtype=I32).cuda()
        self.stack = torch.randperm(150, generator=g).int().cuda()
        self.count = torch.tensor([150], dtype=I32).cuda()
        self.table = torch.zeros(B, 40, dtype=I32).cuda()
        self.cache = torch.full((150, LAYERS, KV, PAGE // 16, 17 * D), 255, dtype=torch.uint8).cuda()
        self.w = [[(1 + 0.2 * torch.randn(D, generator=g)).to(BF16).cuda() for _ in range(2)] for _ in range(LAYERS)]
        a = torch.rand(700, ROT // 2, generator=g) * 6.3
        self.cos_sin = torch.cat([a.cos(), a.sin()], -1).cuda()

    def step(self, q_lens, qkv, most):
        """qkv [LAYERS, T, (HEADS + 2 KV) D] -> [LAYERS, T, HEADS, D]; the loop's own tensors move on."""
        T = qkv.shape[1]
        t = qf.step_tables(self.context, q_lens, self.held, self.table, self.stack, self.count, PAGE, T)
        outs = []
        for layer in range(LAYERS):
            q, k, v = (x.view(T, -1, D) for x in qkv[layer].split([HEADS * D, KV * D, KV * D], -1))
            cache = self.cache[:, layer]
            q, _ = qf.qk_norm_rope(q, k, t.positions, self.cos_sin, *self.w[layer], value=v, cache=cache, slots=t.slots)
            outs.append(qf.kv4_attention(q, cache, t.seq_lens, self.table, D ** -0.5, cu_q=t.cu_q, max_q=most,
                                         out=torch.zeros_like(q)))
        self.context.copy_(t.seq_lens)
        self.held.copy_(t.held)
        self.count.copy_(t.free_count)
        return outs


class Reference:
    def __init__(self, loop):
        self.loop, self.kv = loop, [[(torch.zeros(0, KV, D), torch.zeros(0, KV, D))] * B for _ in range(LAYERS)]

    def step(self, q, qkv):
        cu = [0]
        for n in q:
            cu.append(cu[-1] + n)
        first = [len(self.kv[0][b][0]) for b in range(B)]
        pos = torch.cat([first[b] + torch.arange(q[b]) for b in range(B)])
        outs = []
        for layer in range(LAYERS):
            x, k, v = (t.view(qkv.shape[1], -1, D)[:cu[-1]] for t in qkv[layer].split([HEADS * D, KV * D, KV * D], -1))
            (x, _), (k, _) = (H.norm_rope(t, w.cpu(), 0.0, 1e-6, self.loop.cos_sin.cpu(), pos, False) for t, w in zip((x, k), self.loop.w[layer]))
            k, v = H.rounded(k.float().to(BF16)), H.rounded(v)
            for b in range(B):
                old = self.kv[layer][b]
                self.kv[layer][b] = tuple(torch.cat([o, t[cu[b]:cu[b + 1]]]) for o, t in zip(old, (k, v)))
            keys, vals = zip(*self.kv[layer])
            outs.append((x, keys, vals, cu, [len(t) for t in keys]))
        return outs

    def check(self, got, want):
        for o, (x, keys, vals, cu, seq) in zip(got, want):
            # the query itself is rounded to bf16 (half a step; a step where the fp32 result falls on the other side), which
            # moves a score by at most 2^-7 of the sum of its products' magnitudes
            ref, slack = H.attention(x.float().to(BF16), keys, vals, cu, seq, D ** -0.5)
            H.near(o[:cu[-1]], ref, slack + 2.0 ** -8 * ref.abs().amax(-1, keepdim=True))
            assert not o[cu[-1]:].any()


def _qkv(g, T):
    return torch.randn(LAYERS, T, (HEADS + 2 * KV) * D, generator=g).to(BF16)


def test_a_serving_loop():
    g = H.gen(1)
    loop = Loop(2)
    ref = Reference(loop)
    for step, q in enumerate(([70, 3, 0, 129, 17], [1, 1, 1, 1, 1], [5, 1, 40, 5, 2], [1, 0, 1, 1, 4], [3, 3, 3, 3, 3])):
        qkv = _qkv(g, sum(q) + step)
        got = loop.step(torch.tensor(q, dtype=I32).cuda(), qkv.cuda(), max(q))
        ref.check(got, ref.step(q, qkv))


def test_a_captured_step():
    """A padded step captured once and replayed for other lengths, with eager work and other tensors' frees in between."""
    g = H.gen(3)
    loop = Loop(4)
    ref = Reference(loop)
    T = 16
    q_lens, qkv = torch.zeros(B, dtype=I32).cuda(), _qkv(g, T).cuda()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        loop.step(q_lens, qkv, 4)  # no tokens: nothing moves
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = loop.step(q_lens, qkv, 4)
    start = ([30, 1, 9, 64, 2], _qkv(g, 106))
    ref.check(loop.step(torch.tensor(start[0], dtype=I32).cuda(), start[1].cuda(), 64), ref.step(*start))
    for q in ([1, 1, 1, 1, 1], [4, 0, 4, 4, 4], [2, 3, 1, 0, 4], [1, 4, 4, 3, 1]):
        new = _qkv(g, T)
        qkv.copy_(new)
        q_lens.copy_(torch.tensor(q, dtype=I32))
        graph.replay()
        torch.cuda.synchronize()
        ref.check(out, ref.step(q, new))
        torch.randn(1 << 16, device="cuda").sum().item()


def test_a_step_that_does_not_fit_moves_nothing():
    loop = Loop(5)
    g = H.gen(6)
    loop.step(torch.tensor([9, 9, 9, 9, 9], dtype=I32).cuda(), _qkv(g, 45).cuda(), 9)
    before = [t.clone() for t in (loop.context, loop.held, loop.count, loop.table, loop.cache)]
    out = loop.step(torch.tensor([9, 9, 9, 9, 9], dtype=I32).cuda(), _qkv(g, 44).cuda(), 9)
    assert not any(o.any() for o in out)
    assert all(torch.equal(a, b) for a, b in zip(before, (loop.context, loop.held, loop.count, loop.table, loop.cache)))


def test_bf16_pages_with_the_verification_attention():
    """qk_norm_rope's bf16 pages as gqa_packed_spec_attention reads them."""
    g = H.gen(7)
    T, n = 3, 90
    qkv = torch.randn(n, (8 + 2 * 2) * 128, generator=g).to(BF16)
    q, k, v = (x.view(n, -1, 128) for x in qkv.cuda().split([8 * 128, 256, 256], -1))
    a = torch.rand(n, 32, generator=g) * 6.3
    cos_sin = torch.cat([a.cos(), a.sin()], -1)
    pages = [torch.zeros(8, 16, 2, 128, dtype=BF16, device="cuda") for _ in range(2)]
    order = torch.randperm(8, generator=g)[:6]
    slots = order[torch.arange(n) // 16] * 16 + torch.arange(n) % 16
    x, _ = qf.qk_norm_rope(q, k, torch.arange(n).cuda(), cos_sin.cuda(), value=v, cache=tuple(pages), slots=slots.cuda())
    out = torch.zeros(T, 8, 128, dtype=BF16, device="cuda")
    spec_attn.gqa_packed_spec_attention(x[n - T:].contiguous(), *pages, out, torch.tensor([n], dtype=I32).cuda(),
                                        order[None].int().cuda(), 1, T, 2, 128 ** -0.5)
    (kw, _) = H.norm_rope(k.cpu(), None, 0.0, 0.0, cos_sin, torch.arange(n), False)
    want, slack = H.attention(x[n - T:].cpu(), [kw.float().to(BF16).double()], [v.cpu().double()], [0, T], [n], 128 ** -0.5)
    H.near(out, want, slack + 2.0 ** -7 * want.abs().amax(-1, keepdim=True))
