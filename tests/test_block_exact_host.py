"""That the integer products of exact_cases would show a lost block and a sum kept in 16 bits, and that they take every
form of the kernels (by what the entry points would launch, without a GPU)."""
import random

import pytest
import torch

import block_helpers as H
import exact_cases as X
import launches


def _recorded(kind, cases):
    calls = [(kind, *c) for c in cases]
    return dict(zip(cases, zip(calls, launches.record(calls))))


@pytest.fixture(scope="module")
def plans():
    return _recorded("decode", X.DECODE), _recorded("w8a8", X.W8A8)


def test_every_form_is_taken(plans):
    rng = random.Random(3)
    size = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    decode = [(rng.randint(0, 1), rng.randint(1, 16), size(1, 40000), 64 * size(1, 1000)) for _ in range(40000)]
    w8a8 = [(rng.randint(0, 1), size(1, 3000), size(1, 40000), 64 * size(1, 300)) for _ in range(20000)]
    w8a8 += [(rng.randint(0, 1), size(250, 3000), size(1500, 40000), 64 * size(8, 300)) for _ in range(20000)]
    for kind, sizes, form, own in (("decode", decode, launches.decode_form, plans[0]), ("w8a8", w8a8, launches.w8a8_form, plans[1])):
        sizes = list(dict.fromkeys(c for c in sizes if c[2] * c[3] <= 3e8))
        reached = {form(*r) for r in _recorded(kind, sizes).values()}
        taken = {form(*r) for r in own.values()}
        assert not reached - taken, f"{kind} forms without a case: {sorted(reached - taken)}"


def _columns(N):
    return sorted({n for n in (0, 1, 15, 16, 127, 128, N // 2, N - 2, N - 1) if 0 <= n < N})


def _parts(M, N, K, a8):
    """fp64 [blocks of K, some rows, some channels]: what each block of K adds; and their bias."""
    x, q, s, bias, xd = X.product(M, N, K, a8)
    rows, cols = torch.tensor(sorted({0, M // 2, M - 1})), torch.tensor(_columns(N))
    kb = H.blocks(K)
    xp, qp = torch.zeros(len(rows), kb * H.BLOCK, dtype=torch.float64), torch.zeros(len(cols), kb * H.BLOCK, dtype=torch.float64)
    xp[:, :K], qp[:, :K] = xd[rows], q[cols].double()
    p = torch.einsum("mbk,nbk->bmn", xp.view(len(rows), kb, -1), qp.view(len(cols), kb, -1))
    p *= s[cols // H.BLOCK].double().t()[:, None, :]
    y = p.sum(0) + bias[cols].double()
    assert torch.equal(y.float(), X.reference(xd[rows], q, s, bias)[:, cols])
    return p, y.float()


def _splits(p, n):
    """The K splits' sums, by the kernels' shares of the blocks."""
    at = [i * len(p) // n for i in range(n + 1)]
    return [p[a:b].sum(0) for a, b in zip(at, at[1:])]


@pytest.mark.parametrize("a8", [False, True])
def test_faults_would_show(plans, a8):
    bf16 = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    blocks_seen = 0
    for case, (call, recorded) in plans[a8].items():
        _, M, N, K = case
        if N * K > 25e6:
            continue  # the same generator, only larger
        p, y = _parts(M, N, K, a8)
        lost = (p != 0).double().mean((1, 2))
        # at least 3 outputs are looked at; a block's sum of 64 products or more is zero in one of 12 at most
        assert (lost > 0).all() and lost.mean() > 0.85, case
        blocks_seen += len(p)
        n = launches.w8a8_splits(call, recorded)[2] if a8 else launches.decode_splits(call, recorded)
        if n > 1:
            parts = _splits(p, n)
            exact = sum(parts)
            assert (sum(bf16(t) for t in parts) != exact).any(), case
            for half in range(n):  # a split taken twice, or left out
                assert (parts[half] != 0).any(), case
    assert blocks_seen > 400
