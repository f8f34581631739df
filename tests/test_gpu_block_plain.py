"""The short way of the block-scaled operators' calls (_qf_block_call): it takes a call in its plain form only.  Each of these
calls differs from one that it takes in a single argument; it has to leave it to the long way, which copies or refuses."""
import pytest
import torch

import block_helpers as H

pytestmark = pytest.mark.gpu
BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


class Sub(torch.Tensor):
    pass


def _sub(t):
    return t.as_subclass(Sub)


def _offset(t, n=1):
    """The same values, n elements off their alignment."""
    flat = torch.zeros(t.numel() + 16, dtype=t.dtype, device=t.device)
    v = flat[n:n + t.numel()].view(t.shape)
    v.copy_(t)
    return v


def _padded(t, n):
    """The same values in rows n elements longer."""
    wide = torch.zeros(t.shape[0], t.shape[1] + n, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _columns(t):
    return t.t().contiguous().t()


def _way():
    from qwen_fastpath import _block_lib as B
    from qwen_fastpath.fp8 import _split_workspace
    return (*B.plain(), _split_workspace)


def _no_call(good, take, wrong):
    assert take(good) is not None
    for name, change in wrong:
        args = dict(good)
        args.update(change)
        assert take(args) is None, name


def test_product():
    way, device, stream, workspace = _way()
    g = H.gen(0)
    q, s = H.weight(g, 208, 256)
    q, s, x, bias = q.cuda(), s.cuda(), H.rows(g, 24, 256).cuda(), torch.zeros(208, dtype=BF16, device="cuda")
    bytes_ = q.view(U8)
    fp8 = lambda t: t.view(H.FP8)  # noqa: E731
    good = dict(x=x, w=q.t(), s=s, bias=bias, f32=False, n=-1, decode=-1, device=device)
    take = lambda a: way.product(a["x"], a["w"], a["s"], a["bias"], a["f32"], a["n"], a["decode"], workspace, a["device"], stream)  # noqa: E731
    image = torch.zeros(208 * 256, dtype=U8, device="cuda").view(H.FP8)
    assert take({**good, "w": image}) is not None and take({**good, "w": image, "n": 200, "s": s, "bias": None}) is not None
    _no_call(good, take, [
        ("no tensor", dict(x=3)), ("host x", dict(x=x.cpu())), ("subclass", dict(x=_sub(x))), ("x type", dict(x=x.half())), ("x 3-D", dict(x=x.view(2, 12, 256))),
        ("no rows", dict(x=x[:0])), ("x columns", dict(x=_columns(x))), ("x address", dict(x=_offset(x))), ("x stride", dict(x=_padded(x, 4))),
        ("x overlapping", dict(x=x[:1].expand(24, 256))), ("K not of 64", dict(x=x[:, :200].contiguous())), ("K of another weight", dict(x=x[:, :192].contiguous())),
        ("host w", dict(w=q.cpu().t())), ("w bytes", dict(w=bytes_.t())), ("w rows", dict(w=q)), ("w address", dict(w=fp8(_offset(bytes_)).t())),
        ("w stride", dict(w=fp8(_padded(bytes_, 8)).t())), ("w overlapping", dict(w=q[:1].expand(208, 256).t())), ("w 3-D", dict(w=q.t()[None])),
        ("image short", dict(w=image[:-16])), ("image strided", dict(w=torch.cat([image, image])[::2])), ("image of other channels", dict(w=image, n=192)),
        ("image of none", dict(w=image, n=0)), ("other channels", dict(n=207)), ("host s", dict(s=s.cpu())), ("s type", dict(s=s.double())), ("s shape", dict(s=s[:1])),
        ("s blocks", dict(s=s[:, :1])), ("s 1-D", dict(s=s.view(-1))), ("s strided", dict(s=_columns(s))), ("host bias", dict(bias=bias.cpu())),
        ("bias type", dict(bias=bias.float())), ("bias short", dict(bias=bias[:207])), ("bias strided", dict(bias=torch.cat([bias, bias])[::2])),
        ("bias 2-D", dict(bias=bias[None])), ("too many rows", dict(decode=1)), ("another device", dict(device=device + 1))])
    with pytest.raises(TypeError):
        way.product(x)


def test_norm():
    way, device, stream, _ = _way()
    x, r = torch.ones(6, 64, dtype=BF16, device="cuda"), torch.ones(6, 64, device="cuda")
    w = torch.ones(64, dtype=BF16, device="cuda")
    good = dict(x=x, r=r, post=w, pre=w, gate=x, act=1, eps=1e-6, device=device)
    take = lambda a: way.norm(a["x"], a["r"], a["post"], a["pre"], a["gate"], a["act"], 1.0, a["eps"], 0.0, a["device"], stream)  # noqa: E731
    for gate in (None, w, x[:, :1], x):
        assert take({**good, "gate": gate}) is not None
    _no_call(good, take, [
        ("host x", dict(x=x.cpu())), ("subclass", dict(x=_sub(x))), ("x type", dict(x=x.half())), ("x 1-D", dict(x=x[0])), ("no rows", dict(x=x[:0], r=r[:0], gate=None)),
        ("x columns", dict(x=_columns(x))), ("x address", dict(x=_offset(x))), ("x stride", dict(x=_padded(x, 4))), ("N", dict(x=x[:, :60].contiguous(), r=r[:, :60].contiguous(), post=None, pre=None, gate=None)),
        ("host r", dict(r=r.cpu())), ("r type", dict(r=r.double())), ("r rows", dict(r=r[:5])), ("r columns", dict(r=r[:, :56])), ("r transposed", dict(r=_columns(r))),
        ("r address", dict(r=_offset(r))), ("r stride", dict(r=_padded(r, 2))), ("post type", dict(post=w.float())), ("post short", dict(post=w[:56])),
        ("post address", dict(post=_offset(w))), ("pre type", dict(pre=w.float())), ("pre short", dict(pre=w[:56])), ("pre address", dict(pre=_offset(w))),
        ("pre strided", dict(pre=torch.cat([w, w])[::2])), ("host gate", dict(gate=x.cpu())), ("gate type", dict(gate=x.float())), ("gate short", dict(gate=w[:56])),
        ("gate rows", dict(gate=x[:5])), ("gate of some columns", dict(gate=x[:, :2])), ("gate transposed", dict(gate=_columns(x))), ("gate address", dict(gate=_offset(x))),
        ("gate stride", dict(gate=_padded(x, 4))), ("gate 3-D", dict(gate=x[None])), ("a token's gates", dict(gate=x[:5, :1])), ("act", dict(act=2)),
        ("eps", dict(eps=-1.0)), ("eps no number", dict(eps=float("nan"))), ("another device", dict(device=device + 1))])
    with pytest.raises(TypeError):
        way.norm(x)


def test_moe():
    way, device, stream, _ = _way()
    E, I, Hd, T = 5, 192, 128, 7
    x, logits = torch.ones(T, Hd, dtype=BF16, device="cuda"), torch.zeros(T, E, device="cuda")
    fp8 = lambda t: t.view(H.FP8)  # noqa: E731
    b13, b2 = torch.zeros(E * 2 * I * Hd, dtype=U8, device="cuda"), torch.zeros(E * Hd * I, dtype=U8, device="cuda")
    s13, s2 = torch.ones(E, 4, 1, device="cuda"), torch.ones(E, 1, 2, device="cuda")
    good = dict(x=x, l=logits, w13=fp8(b13), s13=s13, w2=fp8(b2), s2=s2, k=2, device=device)
    take = lambda a: way.moe(a["x"], a["l"], a["w13"], a["s13"], a["w2"], a["s2"], a["k"], True, a["device"], stream)  # noqa: E731
    assert take({**good, "l": logits.to(BF16)}) is not None
    _no_call(good, take, [
        ("host x", dict(x=x.cpu())), ("subclass", dict(x=_sub(x))), ("x type", dict(x=x.half())), ("x 1-D", dict(x=x[0])), ("no rows", dict(x=x[:0], l=logits[:0])),
        ("too many rows", dict(x=x[:1].repeat(17, 1), l=logits[:1].repeat(17, 1))), ("x columns", dict(x=_columns(x))), ("x address", dict(x=_offset(x))),
        ("x stride", dict(x=_padded(x, 4))), ("x overlapping", dict(x=x[:1].expand(T, Hd))), ("H", dict(x=x[:, :96].contiguous())), ("another H", dict(x=x[:, :64].contiguous())),
        ("host logits", dict(l=logits.cpu())), ("logits type", dict(l=logits.half())), ("logits rows", dict(l=logits[:6])), ("logits 1-D", dict(l=logits[0])),
        ("logits columns", dict(l=_columns(logits))), ("logits overlapping", dict(l=logits[:1].expand(T, E))), ("other experts", dict(l=logits[:, :4].contiguous())),
        ("k 0", dict(k=0)), ("k past the experts", dict(k=6)), ("w13 bytes", dict(w13=b13)), ("w13 2-D", dict(w13=fp8(b13).view(-1, Hd))), ("w13 short", dict(w13=fp8(b13)[:-16])),
        ("w13 address", dict(w13=fp8(_offset(b13)))), ("w13 strided", dict(w13=fp8(torch.cat([b13, b13]))[::2])), ("w2 bytes", dict(w2=b2)), ("w2 2-D", dict(w2=fp8(b2).view(-1, I))),
        ("w2 short", dict(w2=fp8(b2)[:-16])), ("w2 address", dict(w2=fp8(_offset(b2)))), ("w2 strided", dict(w2=fp8(torch.cat([b2, b2]))[::2])),
        ("another I", dict(w2=fp8(b2)[:E * Hd * 128])), ("host w2", dict(w2=fp8(b2.cpu()))), ("s13 type", dict(s13=s13.double())), ("s13 shape", dict(s13=s13[:, :2])),
        ("s13 experts", dict(s13=s13[:4])), ("s13 2-D", dict(s13=s13[..., 0])), ("s13 strided", dict(s13=torch.ones(E, 4, 2, device="cuda")[:, :, :1])),
        ("s2 type", dict(s2=s2.double())), ("s2 shape", dict(s2=s2[:, :, :1])), ("s2 2-D", dict(s2=s2[:, 0])), ("s2 strided", dict(s2=_columns(s2[:, 0])[:, None])),
        ("host s2", dict(s2=s2.cpu())), ("another device", dict(device=device + 1))])
    big = torch.zeros(T, 40, device="cuda")
    w13, w2 = fp8(torch.zeros(40 * 2 * 64 * Hd, dtype=U8, device="cuda")), fp8(torch.zeros(40 * Hd * 64, dtype=U8, device="cuda"))
    many = dict(good, l=big, w13=w13, s13=torch.ones(40, 2, 1, device="cuda"), w2=w2, s2=torch.ones(40, 1, 1, device="cuda"))
    assert take({**many, "k": 16}) is not None and take({**many, "k": 17}) is None
    with pytest.raises(TypeError):
        way.moe(x)
