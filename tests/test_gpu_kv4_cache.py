"""The 4-bit cache's writer and reader, bit for bit against the layout and the quantiser written out in kv4_helpers."""
import pytest
import torch

import kv4_helpers as H
import qwen_fastpath as qf

pytestmark = pytest.mark.gpu
BF16, U8 = torch.bfloat16, torch.uint8


def _rows(g, *shape):
    x = torch.randn(*shape, generator=g) * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=g))
    x[..., ::19] *= 8
    return x.to(BF16)


def _check(cache, before, slots, key, value):
    want = before.clone()
    H.write(want, slots, key, value)
    got = cache.cpu()
    # a code's sign is free where its magnitude is 0
    D = got.shape[-1] // 17
    a, b = got[..., :16 * D], want[..., :16 * D]
    for shift in (0, 4):
        x, y = a >> shift & 15, b >> shift & 15
        assert torch.equal(torch.where(x == 8, 0, x), torch.where(y == 8, 0, y))
    assert torch.equal(got[..., 16 * D:], want[..., 16 * D:])


@pytest.mark.parametrize("D,heads,page,T", [(64, 1, 16, 1), (64, 3, 48, 37), (128, 2, 16, 5), (128, 8, 64, 130), (256, 1, 32, 33),
                                            (256, 4, 16, 3), (128, 5, 528, 19)])
def test_store(D, heads, page, T):
    g = H.gen(D + T)
    k, v = _rows(g, T, heads, D), _rows(g, T, heads, D)
    blocks = -(-T // page) + 2
    before = torch.randint(0, 255, (blocks, heads, page // 16, 17 * D), generator=g, dtype=U8)
    slots = torch.randperm(blocks * page, generator=g)[:T]
    slots[T // 2::7] = torch.tensor([-1, blocks * page, -2 ** 40, 2 ** 62])[torch.arange(len(slots[T // 2::7])) % 4]
    cache = before.cuda()
    qf.kv4_store(k.cuda(), v.cuda(), cache, slots.cuda())
    _check(cache, before, slots, k, v)
    inside = (slots >= 0) & (slots < blocks * page)
    got = qf.kv4_load(cache, slots.cuda())
    for x, y in zip(got, (k, v)):
        assert x.shape == (T, heads, D) and x.dtype is BF16
        assert torch.equal(x.cpu().double(), torch.where(inside[:, None, None], H.rounded(y), 0.0))


def test_every_bf16_value():
    """Blocks of neighbouring bit patterns (all exponents, both signs, subnormal numbers, infinities, NaN)."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16).view(512, 1, 128)
    cache, slots = qf.kv4_cache(32, 16, 1, 128), torch.arange(512).cuda()
    qf.kv4_store(x.cuda(), x.flip(0).cuda(), cache, slots)
    k, v = (t.cpu().double() for t in qf.kv4_load(cache, slots))
    for got, want in ((k, H.rounded(x)), (v, H.rounded(x.flip(0)))):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_ties_and_the_scale():
    """Each border between two codes, and largest magnitudes on both sides of 7 * 2^e, over the exponents."""
    rows = []
    for e in (-120, -30, -1, 0, 1, 40, 120):
        for top in (4.0, 6.0, 6.96875, 7.0, 7.96875):
            x = torch.zeros(32)
            x[0] = top
            x[1:8] = H.BORDERS.float()
            x[8:15] = -H.BORDERS.float()
            x[15:23] = H.GRID.float()
            rows.append(x * 2.0 ** e)
    x = torch.stack(rows)[:, None].repeat(1, 1, 2).to(BF16)
    cache, slots = qf.kv4_cache(5, 16, 1, 64), torch.arange(len(rows)).cuda()
    qf.kv4_store(x.cuda(), x.cuda(), cache, slots)
    for got in qf.kv4_load(cache, slots):
        assert torch.equal(got.cpu().double(), H.rounded(x))


def test_blocks_apart():
    """One layer's blocks of a tensor that holds several layers', and keys that are views of a product's output."""
    g = H.gen(5)
    T, heads, D, page = 21, 2, 128, 16
    whole = torch.randint(0, 255, (4, 3, heads, 1, 17 * D), generator=g, dtype=U8)
    before = whole.clone()
    x = _rows(g, T, 4 * heads, D)
    k, v = x[:, 2:4], x[:, 5:7]
    slots = torch.randperm(4 * page, generator=g)[:T]
    gpu, xg = whole.cuda(), x.cuda()
    qf.kv4_store(xg[:, 2:4], xg[:, 5:7], gpu[:, 1], slots.cuda())
    _check(gpu[:, 1], before[:, 1], slots, k, v)
    assert torch.equal(gpu[:, 0].cpu(), before[:, 0]) and torch.equal(gpu[:, 2].cpu(), before[:, 2])
    got = qf.kv4_load(gpu[:, 1], slots.cuda())
    assert torch.equal(got[0].cpu().double(), H.rounded(k)) and torch.equal(got[1].cpu().double(), H.rounded(v))


def test_slots_past_32_bits():
    """Slots and byte offsets past 2^32 in a cache of more than 2^32 positions of one block size."""
    heads, D, page = 1, 64, 16
    blocks = (2 ** 32 // (17 * D)) + 40  # bytes past 2^32
    cache = torch.empty(blocks, heads, 1, 17 * D, dtype=U8, device="cuda")
    slots = torch.tensor([0, 5, blocks * page - 1, blocks * page - 17, blocks * page])
    cache[torch.div(slots[:4], page, rounding_mode="floor").cuda()] = 0
    x = _rows(H.gen(2), 5, heads, D)
    qf.kv4_store(x.cuda(), x.cuda(), cache, slots.cuda())
    got = qf.kv4_load(cache, slots.cuda())
    want = H.rounded(x)
    want[4] = 0
    assert torch.equal(got[0].cpu().double(), want) and torch.equal(got[1].cpu().double(), want)


def test_copies():
    """Keys whose strides the kernel does not take, slots with a stride, and tensors of a subclass."""
    class Sub(torch.Tensor):
        pass
    x = _rows(H.gen(8), 7, 2, 65)[..., 1:]
    cache = qf.kv4_cache(2, 16, 2, 64)
    slots = torch.arange(14).cuda()[::2]
    qf.kv4_store(x.cuda(), x.cuda().as_subclass(Sub), cache, slots)
    for got in qf.kv4_load(cache, slots):
        assert torch.equal(got.cpu().double(), H.rounded(x))
