"""Inputs and plain 64-bit references of the block-scaled FP8 operators' tests, on the CPU.

Each reference comes with the bound that the operator's arithmetic keeps: a rounding to a type is off by at most half a
step (2^-8 relative for bf16, 2^-24 for fp32), and an fp32 sum of n products by at most n * 2^-23 of the sum of their
magnitudes (each addition rounds, or truncates, by at most 2^-23 of a partial sum that is no larger).  The f8 matrix
instruction adds 8 neighbouring products of a lane at a time, aligned to the largest exponent sum e among them, and drops
what lies below 2^(e - 13): beside 448 * 448 (e = 16) a product of 8 is kept whole and one of 4 is lost, in that group of 8
and in no other.  So each of the other 7 loses less than 2^(e - 13) (the largest, 8 bits long, loses nothing)."""
import torch

BF16 = 2.0 ** -8
F32 = 2.0 ** -24
SUM = 2.0 ** -23
BLOCK = 128
FP8 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // BLOCK)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def weight(g, N, K):
    """Random e4m3 [N, K] over its whole range, with fp32 scales that differ by block."""
    q = (torch.randn(N, K, generator=g) * 90).clamp(-448, 448).to(FP8)
    s = 1e-4 * torch.exp(torch.randn(blocks(N), blocks(K), generator=g))
    return q, s


def widen(q, s):
    N, K = q.shape
    return q.double() * s.double().repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]


def rows(g, M, K):
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
    x[:, ::37] *= 20
    return x.to(torch.bfloat16)


def quantize(x):
    """(q e4m3 [M, K], s fp32 [M, blocks]) from the definition: fp32 quotients, each rounded to nearest even."""
    M, K = x.shape
    f = torch.zeros(M, blocks(K) * BLOCK)
    f[:, :K] = x.float()
    f = f.view(M, -1, BLOCK)
    s = f.abs().amax(-1) / 448.0
    q = torch.where(s[..., None] > 0, f / s[..., None], f).to(FP8)
    return q.view(M, -1)[:, :K].contiguous(), s


def product(x, q, s, bias, a8):
    """(y, bound without the last rounding) of the product in 64 bits; a8: activations quantised."""
    if a8:
        xq, sx = quantize(x)
        xd = xq.double() * sx.double().repeat_interleave(BLOCK, 1)[:, :x.shape[1]]
    else:
        xd = x.double()
    w = widen(q, s)
    y, mag = xd @ w.T, xd.abs() @ w.abs().T
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    # K products and the blocks' scales (three roundings each) in fp32
    bound = (x.shape[1] + 8) * SUM * mag
    return y, bound + dropped(xq, sx, q, s) if a8 else bound


def dropped(xq, sx, q, s):
    """Bound of what the f8 matrix instruction drops of each output: 7 * 2^(e - 13) for every 8 neighbouring k, times the
    block's scales.  On the GPU where there is one: M N K exponents are looked at."""
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    M, K = xq.shape
    N = q.shape[0]
    exponent = lambda v: torch.where(v == 0, -100.0, torch.floor(torch.log2(v.abs())))  # noqa: E731
    ex, ew = exponent(xq.float().to(dev)), exponent(q.float().to(dev))
    ex, ew = (torch.where(torch.isnan(e), 0.0, e) for e in (ex, ew))
    block = torch.arange(K // 8, device=dev) // (BLOCK // 8)
    sw = s.to(dev)[torch.arange(N, device=dev) // BLOCK][:, block]
    out = torch.empty(M, N, dtype=torch.float64)
    step = max(1, (1 << 27) // (N * K))
    for m in range(0, M, step):
        e = ex[m:m + step, None, :] + ew[None]
        e = e.view(*e.shape[:2], K // 8, 8).amax(-1)
        out[m:m + step] = (7 * torch.exp2(e - 13) * sx.to(dev)[m:m + step, None, :][..., block] * sw[None]).sum(-1).double().cpu()
    return out


def within(got, ref, bound, step):
    """Whether got is ref to within `bound` and one rounding of relative size `step` (of what was rounded)."""
    got = got.double().cpu()
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    ok = ~torch.isnan(ref)
    err = (got - ref).abs()[ok]
    limit = (bound + step * (ref.abs() + bound) + 1e-37)[ok]
    worst = (err / limit).max().item() if err.numel() else 0.0
    assert worst <= 1, f"error {worst:.3g} times the bound"


def tiles(q):
    """The TILED image of [N, K] bytes, from its definition."""
    N, K = q.shape
    b = torch.zeros((N + 15) // 16 * 16, K, dtype=torch.uint8)
    b[:N] = q.view(torch.uint8)
    out = torch.empty(b.shape[0] // 16, K // 64, 64, 16, dtype=torch.uint8)
    for lane in range(64):
        out[:, :, lane] = b.view(-1, 16, K // 64, 4, 16)[:, lane % 16, :, lane // 16]
    return out.reshape(-1).view(FP8)
