"""Products whose every partial sum is a whole number below 2^24: exact in fp32 in any order of addition, so the only right
output is one bit pattern.  The values are integers that e4m3 and bf16 hold, the scales powers of two; a block that is lost
or taken twice, a scale of another block, a partial sum kept in 16 bits each change the result.

The sizes take each form of the kernels that plan_decode and plan_tiles reach, at the smallest weights found for it, with
whole and with half last blocks of K, and some longer runs.  (layout, M, N, K), layout 0 row-major, 1 TILED."""
import torch

import block_helpers as H

DECODE = [
    (0, 16, 16654, 1920), (0, 12, 4180, 7808), (0, 3, 17, 64), (0, 4, 17, 5056), (0, 4, 17, 5248), (0, 6, 17, 64),
    (0, 6, 17, 128), (0, 7, 17, 4160), (0, 8, 19, 3968), (0, 15, 17, 64), (0, 16, 17, 128), (0, 14, 18, 2624),
    (0, 16, 17, 2816), (0, 9, 1647, 3904), (0, 10, 1749, 4096), (0, 14, 17, 46720), (0, 15, 17, 47552), (0, 4, 17, 2112),
    (0, 3, 18, 2176), (0, 1, 17, 19776), (0, 3, 17, 19840), (0, 5, 17, 2112), (0, 6, 17, 2176), (0, 5, 17, 18496),
    (0, 7, 17, 19200), (0, 12, 17, 2112), (0, 14, 17, 2176), (0, 15, 17, 19136), (0, 11, 17, 19328), (0, 11, 2099, 4288),
    (0, 9, 2206, 4224), (0, 16, 17, 49472), (0, 10, 17, 49664), (0, 1, 17, 4160), (0, 3, 17, 4352), (0, 4, 17, 50688),
    (0, 3, 17, 56896), (0, 5, 17, 4480), (0, 5, 18, 4288), (0, 8, 17, 49472), (0, 6, 17, 50048), (0, 14, 4170, 2944),
    (0, 16, 477, 33664), (0, 5, 2779, 6912), (0, 5, 402, 59584), (0, 1, 18, 6336), (0, 1, 33, 6400), (0, 1, 869, 24640),
    (0, 5, 1729, 6400), (0, 5, 459, 44544), (0, 9, 17, 3264), (0, 9, 17, 3328), (0, 16, 17, 34304), (0, 11, 17, 35136),
    (1, 10, 21071, 2048), (1, 16, 17, 15168), (1, 13, 17, 15232), (1, 2, 17, 64), (1, 1, 17, 128), (1, 4, 17, 5312),
    (1, 4, 17, 5504), (1, 6, 17, 64), (1, 5, 17, 128), (1, 8, 17, 3968), (1, 8, 17, 4032), (1, 10, 17, 64), (1, 14, 17, 128),
    (1, 16, 17, 2560), (1, 15, 17, 2624), (1, 11, 8680, 3904), (1, 11, 17, 25856), (1, 13, 17, 27072), (1, 4, 17, 2112),
    (1, 2, 17, 2176), (1, 3, 17, 18560), (1, 1, 17, 18752), (1, 6, 17, 2112), (1, 5, 18, 2176), (1, 6, 17, 20544),
    (1, 6, 17, 20992), (1, 10, 17, 2112), (1, 15, 17, 2176), (1, 13, 17, 21248), (1, 14, 17, 21440), (1, 9, 2375, 4800),
    (1, 9, 2508, 4736), (1, 9, 278, 60416), (1, 2, 17, 4160), (1, 2, 17, 4224), (1, 1, 17, 57536), (1, 4, 18, 55296),
    (1, 5, 17, 4224), (1, 5, 18, 4160), (1, 5, 19, 62400), (1, 5, 40, 62464), (1, 10, 1378, 4224), (1, 10, 1487, 4288),
    (1, 9, 257, 55744), (1, 1, 18, 6208), (1, 1, 21, 6272), (1, 1, 1077, 18816), (1, 5, 1485, 6272), (1, 5, 1660, 6720),
    (1, 6, 455, 49536), (1, 11, 4122, 4352), (1, 9, 898, 30784), (1, 16, 5120, 17408), (1, 5, 5120, 25600),
    (1, 7, 810, 35072), (1, 16, 31478, 2688), (0, 16, 2498, 14848), (0, 9, 480, 50304), (1, 9, 480, 50304),]

W8A8 = [
    (0, 387, 33623, 576), (0, 274, 33495, 1728), (0, 1, 16449, 64), (0, 420, 35326, 704), (0, 1, 9561, 3328),
    (0, 279, 34581, 3584), (0, 69, 17574, 64), (0, 515, 26143, 896), (0, 65, 9340, 5312), (0, 265, 37768, 4800),
    (0, 130, 37873, 64), (0, 578, 6582, 4992), (0, 2183, 9276, 4864), (1, 392, 33816, 576), (1, 295, 32935, 1920),
    (1, 1, 16610, 64), (1, 396, 35602, 704), (1, 1, 8759, 4032), (1, 294, 34510, 3264), (1, 84, 16385, 64),
    (1, 513, 26452, 832), (1, 71, 8964, 4160), (1, 275, 37589, 5056), (1, 130, 34023, 64), (1, 455, 8262, 4800),
    (1, 709, 27282, 4800), (0, 17, 33, 192), (1, 63, 130, 320), (0, 77, 2500, 2112), (1, 300, 130, 8256),
    (0, 904, 663, 11648), (0, 532, 588, 9600), (1, 904, 663, 11648), (1, 532, 588, 9600),]


def ints(g, top, *shape):
    return torch.randint(-top, top + 1, shape, generator=g, dtype=torch.int8)


def product(M, N, K, a8, seed=0):
    """(x bf16, q e4m3, s fp32, bias bf16, xd fp64 the values that are multiplied): |x q| summed with its scales is at most
    112 K (decode) or 11232 a block (a8), the bias 64."""
    g = H.gen(seed + 7 * M + 5 * N + K)
    nb, kb = H.blocks(N), H.blocks(K)
    s = 2.0 ** torch.randint(0, 2, (nb, kb), generator=g)
    bias = ints(g, 64, N).to(torch.bfloat16)
    if not a8:
        assert 112 * K + 64 < 2 ** 24
        x, q = ints(g, 7, M, K).to(torch.bfloat16), ints(g, 8, N, K).float().to(H.FP8)
        return x, q, s, bias, x.double()
    # a 448 somewhere in each block makes a token's scale 1, times 1, 2 or 4; the quotients are the integers again.  (The f8
    # instruction keeps them: beside 448 * 2 what lies below 2^-4 is dropped.)
    assert 11232 * kb + 64 < 2 ** 24
    x = ints(g, 2, M, K).double()
    x[:, torch.arange(kb) * H.BLOCK + torch.randint(0, 64, (kb,), generator=g)] = 448.0
    x *= (2.0 ** torch.randint(0, 3, (M, kb), generator=g)).double().repeat_interleave(H.BLOCK, 1)[:, :K]
    xb = x.to(torch.bfloat16)
    assert torch.equal(xb.double(), x)
    return xb, ints(g, 2, N, K).float().to(H.FP8), s, bias, x


def reference(xd, q, s, bias):
    """The exact product as fp32, on the tensors' device."""
    N, K = q.shape
    y = torch.empty(xd.shape[0], N, dtype=torch.float64, device=xd.device)
    for n in range(0, N, 4096):  # a few hundred MB of widened weights at once
        at = slice(n, min(N, n + 4096))
        w = q[at].double() * s.double()[n // H.BLOCK:].repeat_interleave(H.BLOCK, 0)[:at.stop - n].repeat_interleave(H.BLOCK, 1)[:, :K]
        y[:, at] = xd @ w.t() + bias[at].double()
    assert y.abs().max() < 2 ** 24
    return y.float()


# ---- experts' layer: (T, E, k, H, I), k a power of two ----
# the routing's kernels; H and I that end in half a block, an odd last tile; second products with and without splits of the
# units; one and two passes over the blocks of H, 4 to 16 wavefronts; one unit a wavefront and many
MOE = [
    (1, 1, 1, 64, 64), (1, 8, 2, 128, 128), (16, 4, 1, 64, 320), (16, 16, 8, 256, 128), (7, 130, 16, 128, 64), (5, 512, 8, 64, 64),
    (3, 300, 4, 128, 192), (16, 65, 2, 1088, 192), (16, 100, 8, 320, 192), (4, 8, 8, 2112, 1344), (9, 20, 16, 64, 1344),
    (2, 3, 2, 4096, 64), (2, 3, 2, 4160, 64), (3, 4, 2, 8192, 192), (16, 40, 8, 2688, 448), (1, 12, 8, 2048, 768),
    (7, 24, 4, 2112, 1344), (16, 24, 8, 2048, 768), (1, 70, 1, 192, 2112), (2, 9, 4, 7168, 320), (6, 10, 2, 512, 64)]


def experts(T, E, k, Hd, I, seed=0):
    """(x bf16, logits fp32, [(q13 e4m3 [2 I, H], s13)], [(q2 e4m3 [H, I], s2)], {token: its experts}) with

    * gate sums about 1024 (1024 from k = 0, the others' sum stays beside it), where silu(g) = g / (1 + exp(-g)) is g in fp32;
    * up sums of at most 12, six values a row, so that an activation is a whole number below 2^15: one bf16 does not hold
      it, the sum of two does;
    * a token's experts equally likely, 1, 2, 4, ... k of them, so that their weights are powers of two.

    W2 is sparse: the sum of all |c w2 a| stays below 2^24 of its unit."""
    g = H.gen(seed + T + 3 * E + 5 * Hd + 7 * I)
    ib, hb = H.blocks(I), H.blocks(Hd)
    x = ints(g, 1, T, Hd).to(torch.bfloat16)
    x[:, 0] = 8.0
    up, down = [], []
    for _ in range(E):
        gate, ups = ints(g, 1, I, Hd), torch.zeros(I, Hd, dtype=torch.int8)
        gate[:, 0] = 0
        gate = gate.float()
        gate[:, 0] = 128.0
        ups.scatter_(1, torch.randint(1, Hd, (I, 6), generator=g), (2 * torch.randint(0, 2, (I, 6), generator=g) - 1).to(torch.int8))
        s = 2.0 ** torch.randint(0, 2, (2 * ib, hb), generator=g)
        s[:ib, 0] = 1.0
        up.append((torch.cat([gate, ups.float()]).to(H.FP8), s))
        w2 = ints(g, 2, Hd, I) * (torch.rand(Hd, I, generator=g) < 0.06)
        down.append((w2.float().to(H.FP8), 2.0 ** torch.randint(0, 2, (hb, ib), generator=g)))
    logits, chosen = torch.full((T, E), -float("inf")), {}
    for t in range(T):
        n = 2 ** int(torch.randint(0, k.bit_length(), (1,), generator=g)) if t % 3 == 2 else k
        chosen[t] = sorted(torch.randperm(E, generator=g)[:n].tolist())
        logits[t, chosen[t]] = float(t % 5) - 2.0
    return x, logits, up, down, chosen


def activations(x, q13, s13, without=None):
    """fp64 [I] activations of one token; without: (0 gate or 1 up, block of H) that is left out."""
    I = q13.shape[0] // 2
    ends = []
    for half, rows, scales in ((0, slice(0, I), slice(0, H.blocks(I))), (1, slice(I, 2 * I), slice(H.blocks(I), None))):
        w = H.widen(q13[rows], s13[scales])
        if without is not None and without[0] == half:
            w[:, H.BLOCK * without[1]:H.BLOCK * (without[1] + 1)] = 0
        ends.append(w @ x.double())
    return ends


def layer_units(x, up, down, chosen):
    """{token: (c, fp64 [experts, half blocks of I, 2 (bf16 parts), H])}: what each part adds to y[t] / c."""
    out = {}
    for t, ids in chosen.items():
        c = 1.0 / len(ids)
        units = []
        for e in ids:
            gate, ups = activations(x[t], *up[e])
            assert gate.min() >= 32 and gate.max() < 2048 and ups.abs().max() <= 12
            a = gate * ups
            hi = a.to(torch.bfloat16).double()
            lo = a - hi
            assert torch.equal(lo.to(torch.bfloat16).double(), lo)
            w2 = H.widen(*down[e])
            assert (w2.abs() @ a.abs()).max() * 1.0 < 2 ** 24 / 16  # of up to 16 experts, in units of c
            parts = [(w2 * v).view(w2.shape[0], -1, 64).sum(2).t() for v in (hi, lo)]
            units.append(torch.stack(parts, 1))
        out[t] = c, torch.stack(units)
    return out


def layer(units, T, Hd):
    """y bf16 from layer_units: the exact sums, rounded once."""
    y = torch.zeros(T, Hd, dtype=torch.float64)
    for t, (c, u) in units.items():
        y[t] = c * u.sum((0, 1, 2))
    assert torch.equal(y.float().double(), y)
    return y.float().to(torch.bfloat16)
