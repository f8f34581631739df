"""A whole mixture-of-experts layer for a few tokens (decode, speculative verification) over block-scaled FP8 experts.

Two launches for routing, gate and up products, activation, down product and the weighted sum (qf_moe_few_tokens,
include/qf_block.h): each chosen expert's weights are read once for all its tokens, and nothing comes back to the host,
so the call may be captured in a HIP graph.
"""
from __future__ import annotations

import torch

from . import _block_lib as B
from .fp8 import _rows, fp8_scale_shape
from .w8a16 import tiled_numel

_BF16, _FP8, _F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32


def moe_few_tokens(x: torch.Tensor, router_logits: torch.Tensor, w13: torch.Tensor, s13: torch.Tensor, w2: torch.Tensor,
                   s2: torch.Tensor, top_k: int, renormalize: bool = True) -> torch.Tensor:
    """y[t] = sum over the top_k experts e of token t: c[t, e] * W2_e (silu(Wgate_e x[t]) * (Wup_e x[t])).

    x bf16 [T, H], T <= 16; router_logits bf16 or fp32 [T, E].  c = softmax(logits), divided by the chosen ones' sum with
    ``renormalize``; the largest logits are chosen, the lowest index first among equal ones; a token whose logits are all
    -inf has no expert (zeros: padding rows of a captured batch), and an expert of weight 0 is not read for it.  w13: the
    TILED image (fp8_to_tiled) of the [E * 2 I, H] matrix of each expert's I gate rows, then its I up rows, s13 fp32
    [E, 2 ceil(I / 128), ceil(H / 128)] in that order; w2: the image of [E * H, I], s2 fp32 [E, ceil(H / 128),
    ceil(I / 128)].  H and I multiples of 64; E <= 512, top_k <= min(E, 16).  Activations stay bf16, weights are widened
    exactly, sums are fp32; the activation is kept to 16 bits between the products, y is rounded once at the end."""
    if x.is_cuda:
        plain, device, stream = B.plain()
        y = plain.moe(x, router_logits, w13, s13, w2, s2, int(top_k), renormalize, device, stream)
        if y is not None:
            return y
    if x.dim() != 2 or x.dtype is not _BF16:
        raise TypeError(f"x must be a 2-D bf16 tensor, got {x.dtype} {tuple(x.shape)}")
    if router_logits.dim() != 2 or (router_logits.dtype is not _F32 and router_logits.dtype is not _BF16):
        raise TypeError(f"router_logits must be 2-D bf16 or fp32, got {router_logits.dtype} {tuple(router_logits.shape)}")
    if w13.dtype is not _FP8 or w2.dtype is not _FP8 or s13.dtype is not _F32 or s2.dtype is not _F32:
        raise TypeError("expected float8_e4m3fn weights with fp32 scales")
    dev = B.same_gpu(x, router_logits, w13, s13, w2, s2)
    T, H = x.shape
    E = router_logits.shape[1]
    if T > B.MAX_DECODE_M:
        raise ValueError(f"at most {B.MAX_DECODE_M} tokens, got {T}")
    if router_logits.shape[0] != T or not 1 <= E <= B.MOE_MAX_EXPERTS:
        raise ValueError(f"router_logits must be [{T}, 1..{B.MOE_MAX_EXPERTS}], got {list(router_logits.shape)}")
    top_k = int(top_k)
    if not 1 <= top_k <= min(E, B.MOE_MAX_TOP_K):
        raise ValueError(f"top_k must be in [1, {min(E, B.MOE_MAX_TOP_K)}], got {top_k}")
    if w13.dim() != 1 or w2.dim() != 1 or not w13.is_contiguous() or not w2.is_contiguous():
        raise ValueError("w13 and w2 must be TILED images (fp8_to_tiled)")
    if H < 64 or H % 64:
        raise ValueError(f"H must be a multiple of 64, got {H}")
    I = w2.numel() // (E * H)
    if I < 64 or I % 64 or w2.numel() != tiled_numel(E * H, I) or w13.numel() != tiled_numel(E * 2 * I, H):
        raise ValueError(f"w13 and w2 must be the images of [{E} * 2 I, {H}] and [{E} * {H}, I], I a multiple of 64, got "
                         f"{w13.numel()} and {w2.numel()} bytes")
    nb, kb = fp8_scale_shape(I, H)
    if s13.shape != (E, 2 * nb, kb) or s2.shape != (E, kb, nb):
        raise ValueError(f"s13 and s2 must be {[E, 2 * nb, kb]} and {[E, kb, nb]}, got {list(s13.shape)} and {list(s2.shape)}")
    if w13.data_ptr() % 16 or w2.data_ptr() % 16:
        raise ValueError("w13 and w2 must be 16-byte aligned")
    y = x.new_empty((T, H))
    if T == 0:
        return y
    if not s13.is_contiguous():
        s13 = s13.contiguous()
    if not s2.is_contiguous():
        s2 = s2.contiguous()
    x, ldx = _rows(x)
    if router_logits.stride(1) != 1 or (T > 1 and router_logits.stride(0) < E):
        router_logits = router_logits.clone(memory_format=torch.contiguous_format)
    nbytes = B.workspace_bytes("qf_moe_few_workspace_bytes", T, E, top_k, H, I)
    ws = x.new_empty(nbytes, dtype=torch.uint8)  # the caching allocator's: one a call, capture-safe
    B.call("qf_moe_few_tokens", dev, x.data_ptr(), ldx, router_logits.data_ptr(),
           router_logits.stride(0) if T > 1 else E, router_logits.dtype is _F32, w13.data_ptr(), s13.data_ptr(),
           w2.data_ptr(), s2.data_ptr(), y.data_ptr(), H, T, E, top_k, H, I, bool(renormalize), ws.data_ptr(), nbytes)
    return y
