"""That the integer layers of exact_cases would show an activation kept in one bf16 instead of two, a block of H that is
left out, a unit that is lost; and that they take each form of the two launches (without a GPU)."""
import random

import pytest
import torch

import block_helpers as H
import exact_cases as X
import launches


@pytest.mark.parametrize("T,E,k,Hd,I", X.MOE)
def test_faults_would_show(T, E, k, Hd, I):
    x, logits, up, down, chosen = X.experts(T, E, k, Hd, I)
    units = X.layer_units(x, up, down, chosen)
    y = X.layer(units, T, Hd)
    one_part = {t: (c, u[:, :, :1]) for t, (c, u) in units.items()}
    assert (X.layer(one_part, T, Hd) != y).double().mean() > 0.05
    half_blocks = I // 64
    low_seen = torch.zeros(half_blocks, dtype=torch.bool)
    for t, (c, u) in units.items():
        whole = c * u.sum((0, 1, 2))
        differ = lambda off: (off.float().to(torch.bfloat16) != y[t]).any(-1)  # noqa: E731,B023
        assert differ(whole - c * u.sum(2)).all()  # any expert's half block of I
        low_seen |= differ(whole - c * u[:, :, 1].sum(0))  # the low parts of a half block of I, of the token's experts
    assert low_seen.all()
    c, u = units[0]
    whole = c * u.sum((0, 1, 2))
    w2 = {e: H.widen(*down[e]) for e in chosen[0]}
    a = {e: torch.mul(*X.activations(x[0], *up[e])) for e in chosen[0]}
    for half in (0, 1):  # a block of H, of the gate rows or of the up rows
        for b in range(H.blocks(Hd)):
            off = whole + c * sum(w2[e] @ (torch.mul(*X.activations(x[0], *up[e], without=(half, b))) - a[e]) for e in chosen[0])
            assert (off.float().to(torch.bfloat16) != y[0]).any(), (half, b)


def _form(call, recorded):
    """(the routing's kernel, wavefronts, passes over the blocks of H, splits of the second launch or none)."""
    _, T, E, k, Hd, I = call
    first, second = recorded[2]
    waves = first.threads // 64
    return first.params, -(-H.blocks(Hd) // (2 * waves)) > 1, second.grid[1] > 1


def test_every_form_is_taken():
    rng = random.Random(4)
    size = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    calls = []
    for _ in range(4000):
        E = size(1, 512)
        calls.append(("moe", rng.randint(1, 16), E, rng.randint(1, min(16, E)), 64 * size(1, 40), 64 * size(1, 24)))
    forms = lambda calls: [_form(c, r) for c, r in zip(calls, launches.record(calls))]  # noqa: E731
    reached, taken = forms(calls), forms([("moe", *c) for c in X.MOE])
    for i, what in enumerate(("routing", "passes over H", "splits")):
        assert {f[i] for f in reached} <= {f[i] for f in taken}, what
    assert {(f[1], f[2]) for f in reached} <= {(f[1], f[2]) for f in taken}
