"""The norms around a block of a layer, fused with the block's gate and residual scale, on MI355X.

Between two blocks (attention, feed-forward) a layer normalises the block's output, gates and scales it, adds it to the
residual stream and normalises the sum for the next block; ``block_norm_rows`` does all of it in one launch and one pass
over the data (qf_block_norm_rows, include/qf_block.h).  ``rms_norm_rows`` is the plain unit-RMS norm by itself.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _block_lib as B

_BF16, _F32 = torch.bfloat16, torch.float32


def _fit(t: torch.Tensor, align: int) -> bool:
    """Rows the kernel can address: unit column stride, 16-byte aligned, a row stride that is a multiple of `align`."""
    rows, unit = t.stride()
    return unit == 1 and t.data_ptr() % 16 == 0 and (rows % align == 0 or t.shape[0] == 1)


def _weight(w: Optional[torch.Tensor], N: int, name: str) -> Optional[torch.Tensor]:
    if w is None:
        return None
    if w.dtype is not _BF16 or w.shape != (N,):
        raise TypeError(f"{name} must be bf16 [{N}], got {w.dtype} {list(w.shape)}")
    if (N > 1 and w.stride(0) != 1) or w.data_ptr() % 16:
        w = w.clone(memory_format=torch.contiguous_format)
    return w


def _output(out: Optional[torch.Tensor], like: torch.Tensor, M: int, N: int, align: int, name: str) -> torch.Tensor:
    if out is None:
        return torch.empty_like(like) if like.is_contiguous() else like.new_empty((M, N))
    if out.dtype != like.dtype or tuple(out.shape) != (M, N) or out.device != like.device or not _fit(out, align) or (
            M > 1 and out.stride(0) < N):
        raise ValueError(f"{name} must be a {like.dtype} [{M}, {N}] tensor on {like.device} with unit column stride, 16-byte "
                         f"aligned rows that do not overlap and a row stride that is a multiple of {align}")
    return out


def block_norm_rows(x: torch.Tensor, residual: torch.Tensor, post_weight: Optional[torch.Tensor] = None,
                    pre_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                    gate_act: str = "none", alpha: float = 1.0, eps: float = 1e-6, weight_offset: float = 0.0,
                    y: Optional[torch.Tensor] = None, h: Optional[torch.Tensor] = None):
    """(y, h) of a block's output x and the residual stream, row by row:

        p = x * rsqrt(mean(x^2) + eps) * (weight_offset + post_weight)     (x itself without post_weight)
        y = residual + alpha * act(gate) * p
        h = y * rsqrt(mean(y^2) + eps) * (weight_offset + pre_weight)      (no factor without pre_weight)

    x bf16 [M, N]; residual bf16 or fp32 [M, N]; weights bf16 [N] (weight_offset 1 for checkpoints that store them less
    one); gate bf16 [N] (a channel's), [M, 1] (a token's) or [M, N], gate_act "none" or "sigmoid".  All arithmetic is fp32;
    y is rounded once to the residual's type, h, from y before that rounding, once to bf16.  y may be given as the residual and
    h as x (in place); outputs must not overlap the inputs otherwise.  N % 8 == 0, N <= 32768."""
    act = B.ACTS.get(gate_act)
    if x.is_cuda and y is None and h is None and act is not None:
        plain, device, stream = B.plain()
        yh = plain.norm(x, residual, post_weight, pre_weight, gate, act, alpha, eps, weight_offset, device, stream)
        if yh is not None:
            return yh
    if x.dim() != 2 or x.dtype is not _BF16:
        raise TypeError(f"x must be a 2-D bf16 tensor, got {x.dtype} {tuple(x.shape)}")
    wide = residual.dtype is _F32
    if not wide and residual.dtype is not _BF16:
        raise TypeError(f"residual must be bf16 or fp32, got {residual.dtype}")
    if residual.shape != x.shape:
        raise ValueError(f"residual must be {list(x.shape)}, got {list(residual.shape)}")
    M, N = x.shape
    if N < 8 or N % 8 or N > B.NORM_MAX_N:
        raise ValueError(f"N must be a multiple of 8 up to {B.NORM_MAX_N}, got {N}")
    if act is None:
        raise ValueError(f"gate_act must be one of {sorted(B.ACTS)}, got {gate_act!r}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    dev = B.same_gpu(x, residual, post_weight, pre_weight, gate)
    align = 4 if wide else 8
    y = _output(y, residual, M, N, align, "y")
    h = _output(h, x, M, N, 8, "h")
    if M == 0:
        return y, h
    post_weight, pre_weight = _weight(post_weight, N, "post_weight"), _weight(pre_weight, N, "pre_weight")
    if not _fit(x, 8):
        x = x.clone(memory_format=torch.contiguous_format)
    if not _fit(residual, align):
        residual = residual.clone(memory_format=torch.contiguous_format)
    kind, ldg, gptr = B.GATE_NONE, 0, None
    if gate is not None:
        if gate.dtype is not _BF16:
            raise TypeError(f"gate must be bf16, got {gate.dtype}")
        if gate.shape == (N,):
            kind, gate = B.GATE_CHANNEL, _weight(gate, N, "gate")
        elif gate.shape == (M, 1):
            kind, ldg = B.GATE_TOKEN, gate.stride(0) if M > 1 else 0
        elif gate.shape == (M, N):
            if not _fit(gate, 8):
                gate = gate.clone(memory_format=torch.contiguous_format)
            kind, ldg = B.GATE_FULL, gate.stride(0) if M > 1 else 0
        else:
            raise ValueError(f"gate must be [{N}], [{M}, 1] or [{M}, {N}], got {list(gate.shape)}")
        gptr = gate.data_ptr()
    B.call("qf_block_norm_rows", dev, x.data_ptr(), x.stride(0) if M > 1 else N, residual.data_ptr(),
           residual.stride(0) if M > 1 else N, wide, None if post_weight is None else post_weight.data_ptr(),
           None if pre_weight is None else pre_weight.data_ptr(), weight_offset, gptr, ldg, kind, act, alpha, eps, M, N,
           y.data_ptr(), y.stride(0) if M > 1 else N, h.data_ptr(), h.stride(0) if M > 1 else N)
    return y, h
