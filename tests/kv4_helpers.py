"""Plain 64-bit references of the 4-bit cache's operators, on the CPU, and the bounds that their arithmetic keeps.

A rounding to a type is off by at most half a step (2^-8 relative for bf16), an fp32 sum of n products by at most n * 2^-23 of
the sum of their magnitudes.  What is held in 4 bits has to be equal: keys are computed in 64 bits on both sides."""
import math

import torch

BF16, F32 = 2.0 ** -8, 2.0 ** -23
GRID = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
BORDERS = (GRID[1:] + GRID[:-1]) / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def quantise(x):
    """(codes uint8 [..., D], scale bytes uint8 [..., D / 32]) of bf16 values, from the definition."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    bad = ~b.isfinite().all(-1)
    top = torch.where(bad, 1.0, top)
    e = torch.full(top.shape, -125, dtype=torch.int64)
    for _ in range(260):  # the smallest exponent with the largest magnitude below 7 * 2^e
        e += ((top >= 7 * torch.exp2(e.double())) & (e < 125)).long()
    y = torch.where(bad[..., None], 0.0, b) / torch.exp2(e.double())[..., None]
    code = torch.bucketize(y.abs(), BORDERS)  # a border itself: the lower code
    tie = (y.abs()[..., None] == BORDERS).any(-1)
    code = torch.where(tie & (code % 2 == 1), code + 1, code)
    code = (code + 8 * (y < 0).long()).flatten(-2)
    return code.to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


def values(codes, scales):
    """What they stand for, in 64 bits."""
    v = GRID[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)
    s = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def rounded(x):
    """bf16 values as their 4-bit form's, in 64 bits."""
    return values(*quantise(x))


def write(cache, slots, key, value):
    """The tokens' bytes put into a cache uint8 [blocks, heads, page / 16, 17 D] on the CPU, byte by byte as the layout says."""
    _, heads, tiles, record = cache.shape
    D, page = record // 17, tiles * 16
    w = min(D, 128) // 16
    (kc, ks), (vc, vs) = quantise(key), quantise(value)
    d = torch.arange(0, D, 2)
    g = torch.arange(D // 32)
    for t, s in enumerate(slots.tolist()):
        if not 0 <= s < cache.shape[0] * page:
            continue
        block, p = divmod(s, page)
        rec, q = cache[block, :, p // 16], p % 16
        rec[:, q * (D // 2) + d // 2] = kc[t][:, 0::2] | kc[t][:, 1::2] << 4
        half, inside = d // (16 * w), d % (16 * w)
        rec[:, 8 * D + half * 128 * w + ((q // 4 * 16 + inside // w) * 4 + q % 4) * (w // 2) + inside % w // 2] = (
            vc[t][:, 0::2] | vc[t][:, 1::2] << 4)
        rec[:, 16 * D + g * 16 + q] = ks[t]
        rec[:, 16 * D + D // 2 + g * 16 + q] = vs[t]


def norm_rope(x, weight, offset, eps, cos_sin, positions, interleaved):
    """(result, bound on an fp32 computation of it before its rounding) in 64 bits, of [T, H, D]."""
    n = x.double()
    if weight is not None:
        n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + eps) * (offset + weight.double())
    y, size = n.clone(), n.abs()
    if cos_sin is not None:
        rot = cos_sin.shape[1]
        cs = cos_sin.double()[positions.clamp(0, len(cos_sin) - 1)][:, None]
        i = torch.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = cs[..., :rot // 2], cs[..., rot // 2:]
        y[..., a] = n[..., a] * c - n[..., b] * s
        y[..., b] = n[..., b] * c + n[..., a] * s
        size = size.clone()
        size[..., a] = (n[..., a] * c).abs() + (n[..., b] * s).abs()
        size[..., b] = (n[..., b] * c).abs() + (n[..., a] * s).abs()
    # the mean's sum, its root and quotient, the weight's sum, two products and an addition
    return y, (x.shape[-1] + 8) * F32 * size


def near(got, want, slack, what=""):
    """Every value within half a bf16 step of one that is within `slack` of `want`; NaN and infinities where they are."""
    got, want = got.double().cpu(), want.double()
    odd = ~want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    assert torch.equal(got[odd & ~want.isnan()], want[odd & ~want.isnan()]), what
    off = (got - want).abs()[~odd]
    most = (slack + BF16 * (want.abs() + slack))[~odd] + 2.0 ** -133
    assert bool((off <= most).all()), f"{what}: off by {float((off / most).max()):.2f} of the bound"


def attention(query, key, value, cu, seq, scale):
    """(result, bound before its rounding) of [T, H, D] queries over requests' keys and values (lists of [L, H_kv, D], 64 bits).

    The weights' rounding to bf16 is 2^-8 of each; a score is off by its fp32 sum of D exact products, the scale's product and
    the exponent's argument; a sum over L positions, and the splits' factors, by (L + 16) 2^-23.  A weight is held beside the row's
largest, which is 1 or more: one below 2^-126, the smallest normal number, may vanish, in a split or where splits are joined."""
    T, H, D = query.shape
    out, slack = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    for b in range(len(seq)):
        lo, hi, L = int(cu[b]), int(cu[b + 1]), int(seq[b])
        if hi == lo or L == 0:
            continue
        k, v = key[b][:L].double(), value[b][:L].double()
        G = H // k.shape[1]
        last = L - (hi - lo) + torch.arange(hi - lo)
        seen = torch.arange(L) <= last[:, None]
        for h in range(H):
            q, kh, vh = query[lo:hi, h].double(), k[:, h // G], v[:, h // G]
            s = torch.where(seen, q @ kh.t() * scale, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if not s.isnan().any() else torch.softmax(s, -1)
            p = torch.where(seen, p, 0.0)
            # a NaN that a row does not see is no part of it
            clean = torch.nan_to_num(vh, nan=0.0)
            poison = (seen.double() @ vh.isnan().double()) > 0
            out[lo:hi, h] = torch.where(poison, math.nan, p @ clean)
            size = torch.where(seen, (q.abs() @ torch.nan_to_num(kh).abs().t()) * abs(scale), 0.0).amax(-1, keepdim=True)
            score = (D + 4) * F32 * size
            slack[lo:hi, h] = (BF16 + 2 * score + (L + 16) * F32) * (p @ clean.abs()) + 2.0 ** -125 * (seen.double() @ clean.abs())
        out[lo:hi][last < 0] = 0.0
    return out, torch.nan_to_num(slack)


def tables(context, q, held, table, stack, count, page, tokens):
    """step_tables in Python: a dict of lists, and the table changed in place."""
    context, q, held = context.tolist(), q.tolist(), held.tolist()
    width = table.shape[1]
    seq = [c + n for c, n in zip(context, q)]
    need = [max(0, -(-s // page) - h) for s, h in zip(seq, held)]
    fits = (min(context) >= 0 and min(q) >= 0 and min(held) >= 0 and max(held) <= width and sum(q) <= tokens and sum(need) <= count
            and 0 <= count <= len(stack) and max(seq) < 2 ** 31 and all(h + n <= width for h, n in zip(held, need)))
    if not fits:
        return dict(cu_q=[0] * (len(q) + 1), seq_lens=context, positions=[0] * tokens, slots=[-1] * tokens, held=held,
                    free_count=[count], fits=[0])
    cu, positions, slots = [0], [], []
    for b, n in enumerate(q):
        for j in range(need[b]):
            count -= 1
            table[b, held[b] + j] = stack[count]
        cu.append(cu[-1] + n)
        for p in range(context[b], seq[b]):
            positions.append(p)
            slots.append(int(table[b, p // page]) * page + p % page)
    rest = tokens - cu[-1]
    return dict(cu_q=cu, seq_lens=seq, positions=positions + [0] * rest, slots=slots + [-1] * rest,
                held=[h + n for h, n in zip(held, need)], free_count=[count], fits=[1])


def paged(g, lengths, page, spare=2):
    """(number of blocks, int32 table) of requests of these lengths, pages shuffled; entries past a request's are out of range."""
    counts = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(counts) + spare, generator=g)
    table = torch.full((len(lengths), max(1, *counts)), 2 ** 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n].int()
        at += n
    return len(order), table


def slots_of(table, b, length, page):
    at = torch.arange(length)
    return table[b].long()[at // page] * page + at % page
