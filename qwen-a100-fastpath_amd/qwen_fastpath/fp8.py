"""Linear layers of a block-scaled FP8 checkpoint on MI355X: e4m3 weights with one fp32 scale for each 128 x 128 block.

W[n, k] = q[n, k] * scale[n // 128, k // 128].  The two products follow the rule of the int8 layers: up to
MAX_DECODE_M = 16 rows the activations stay bf16 (``fp8_w8a16_mm``: exact products, fp32 sums, bound by the weights'
bytes), above they are quantised to e4m3 per token and block of 128 (``fp8_w8a8_mm``, on the f8 MFMA).  ``fp8_linear``
picks between them.  Weights are the checkpoint's row-major [N, K] matrix, handed over as its [K, N] view with stride
(1, K) as the int8 layers' are, or the TILED image of the same bytes made by ``fp8_to_tiled``, which streams fastest.
The compute is hand-written HIP for gfx950 behind a C ABI (include/qf_block.h); calls run on torch's current stream of
the tensors' device and may be captured in a HIP graph.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _block_lib as B
from .w8a16 import ROWMAJOR, TILED, _workspace, from_tiled, tiled_numel, to_tiled

_MAX_STRIDE = 1 << 26  # longest row stride the products address
_BF16, _FP8, _F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32


def fp8_scale_shape(N: int, K: int) -> tuple[int, int]:
    """Shape of the scales of an [N, K] weight: one for each block of 128 x 128, the last ones maybe of part of a block."""
    return -(-N // B.BLOCK), -(-K // B.BLOCK)


def fp8_to_tiled(w_t: torch.Tensor) -> torch.Tensor:
    """The TILED image (to_tiled) of a [K, N] stride-(1, K) e4m3 weight: ceil(N / 16) * 16 * K bytes, 1-D."""
    if w_t.dtype != _FP8:
        raise TypeError(f"weight must be float8_e4m3fn, got {w_t.dtype}")
    return to_tiled(w_t.view(torch.int8)).view(_FP8)


def fp8_from_tiled(image: torch.Tensor, N: int, K: int) -> torch.Tensor:
    """Inverse of fp8_to_tiled: the [K, N] stride-(1, K) view of a fresh [N, K] matrix."""
    if image.dtype != _FP8:
        raise TypeError(f"image must be float8_e4m3fn, got {image.dtype}")
    if not image.is_contiguous() or image.numel() != tiled_numel(N, K):
        raise ValueError(f"the image of a [{N}, {K}] weight is a contiguous tensor of {tiled_numel(N, K)} bytes")
    return from_tiled(image.view(torch.int8), N, K).view(_FP8)


def quantize_tokens_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 values and fp32 scales of a bf16 [M, K] matrix, a scale for each row and block of 128 values: s = max|x| / 448,
    q = e4m3(x / s), both rounded to nearest even; a block of zeros has scale 0.  K % 64 == 0.  Returns (q [M, K],
    s [M, ceil(K / 128)]): the activations fp8_w8a8_mm multiplies."""
    if x.dim() != 2 or x.dtype != _BF16:
        raise TypeError(f"x must be a 2-D bf16 tensor, got {x.dtype} {tuple(x.shape)}")
    dev = B.same_gpu(x)
    M, K = x.shape
    if K < 64 or K % 64:
        raise ValueError(f"K must be a multiple of 64, got {K}")
    x, ldx = _rows(x)
    q = x.new_empty((M, K), dtype=_FP8)
    s = x.new_empty((M, -(-K // B.BLOCK)), dtype=_F32)
    if M:
        B.call("qf_quantize_tokens_fp8", dev, x.data_ptr(), ldx, M, K, q.data_ptr(), K, s.data_ptr())
    return q, s


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """x with rows the kernels can read (unit column stride, 16-byte aligned, a row stride that is a multiple of 8), and
    the row stride."""
    M, K = x.shape
    ld = x.stride(0) if M > 1 else K
    if (x.stride(1) != 1 and K > 1) or x.data_ptr() % 16 or ld % 8 or not K <= ld <= _MAX_STRIDE:
        return x.clone(memory_format=torch.contiguous_format), K
    return x, ld


def _split_workspace(x: torch.Tensor, nbytes: int) -> torch.Tensor:
    return _workspace(x.device, nbytes)


def _product(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor], out_dtype,
             out_features: Optional[int], decode: Optional[bool]) -> torch.Tensor:
    if x.is_cuda and (out_dtype is _BF16 or out_dtype is _F32):
        plain, device, stream = B.plain()
        y = plain.product(x, w, w_scale, bias, out_dtype is _F32, -1 if out_features is None else max(int(out_features), 0),
                          -1 if decode is None else decode, _split_workspace, device, stream)
        if y is not None:
            return y
    if x.dim() != 2 or x.dtype is not _BF16:
        raise TypeError(f"x must be a 2-D bf16 tensor, got {x.dtype} {tuple(x.shape)}")
    if w.dtype is not _FP8 or w_scale.dtype is not _F32:
        raise TypeError(f"expected float8_e4m3fn weights with fp32 scales, got {w.dtype} and {w_scale.dtype}")
    if out_dtype is not _BF16 and out_dtype is not _F32:
        raise TypeError(f"out_dtype must be bf16 or fp32, got {out_dtype}")
    dev = B.same_gpu(x, w, w_scale, bias)
    M, K = x.shape
    if K < 64 or K % 64:
        raise ValueError(f"K must be a multiple of 64, got {K}")
    if w.dim() == 1:
        layout, ldw = TILED, K
        N = w.numel() // K if out_features is None else int(out_features)
        if N < 1 or not w.is_contiguous() or w.numel() != tiled_numel(N, K):
            raise ValueError(f"the TILED image of a [{N}, {K}] weight is a contiguous tensor of {tiled_numel(N, K)} bytes, "
                             f"got {w.numel()}")
    else:
        layout = ROWMAJOR
        if w.dim() != 2 or w.shape[0] != K or w.stride(0) != 1:
            raise ValueError(f"row-major weight must be a [{K}, N] view with stride(0) == 1, got shape {tuple(w.shape)} "
                             f"stride {w.stride()}")
        N = w.shape[1]
        if N < 1 or (out_features is not None and out_features != N):
            raise ValueError(f"weight has {N} output channels, out_features is {out_features}")
        ldw = w.stride(1) if N > 1 else K
        if not K <= ldw <= _MAX_STRIDE or ldw % 16:
            raise ValueError(f"row-major weight needs a row stride from K to 2^26 that is a multiple of 16, got {ldw}")
    if w.data_ptr() % 16:
        raise ValueError("weight must be 16-byte aligned")
    if w_scale.dim() != 2 or w_scale.shape != fp8_scale_shape(N, K):
        raise ValueError(f"w_scale must be {list(fp8_scale_shape(N, K))}, got {list(w_scale.shape)}")
    if not w_scale.is_contiguous():
        w_scale = w_scale.contiguous()
    if bias is not None:
        if bias.dtype is not _BF16 or bias.shape != (N,):
            raise TypeError(f"bias must be bf16 [{N}], got {bias.dtype} {list(bias.shape)}")
        if not bias.is_contiguous():
            bias = bias.contiguous()
    y = x.new_empty((M, N), dtype=out_dtype)
    if M == 0:
        return y
    x, ldx = _rows(x)
    args = (x.data_ptr(), ldx, w.data_ptr(), ldw, layout, w_scale.data_ptr(), None if bias is None else bias.data_ptr(),
            y.data_ptr(), N, 0 if out_dtype is _BF16 else 1, M, N, K)
    if M <= B.MAX_DECODE_M if decode is None else decode:
        nbytes = B.workspace_bytes("qf_fp8_w8a16_workspace_bytes", M, N, K, layout)
        ws = _workspace(x.device, nbytes) if nbytes else None  # K splits' arrival counters: zero between calls
        B.call("qf_fp8_w8a16_gemm", dev, *args, None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel())
    else:
        nbytes = B.workspace_bytes("qf_fp8_w8a8_workspace_bytes", M, N, K)
        ws = x.new_empty(nbytes, dtype=torch.uint8)  # the caching allocator's: one a call, capture-safe
        B.call("qf_fp8_w8a8_linear", dev, *args, ws.data_ptr(), nbytes)
    return y


def fp8_w8a16_mm(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, out_dtype: torch.dtype = _BF16,
                 bias: Optional[torch.Tensor] = None, out_features: Optional[int] = None) -> torch.Tensor:
    """y[M, N] = x @ W^T (+ bias) with bf16 activations, M <= 16: exact products, fp32 sums, one rounding to out_dtype.
    x bf16 [M, K], K % 64 == 0; w the [K, N] stride-(1, K) e4m3 view or a TILED image (out_features = N where that is not
    a multiple of 16); w_scale fp32 [ceil(N / 128), ceil(K / 128)]; bias bf16 [N]."""
    if x.dim() == 2 and x.shape[0] > B.MAX_DECODE_M:
        raise ValueError(f"at most {B.MAX_DECODE_M} rows, got {x.shape[0]}: fp8_w8a8_mm serves more")
    return _product(x, w, w_scale, bias, out_dtype, out_features, True)


def fp8_w8a8_mm(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, out_dtype: torch.dtype = _BF16,
                bias: Optional[torch.Tensor] = None, out_features: Optional[int] = None) -> torch.Tensor:
    """y[M, N] = xq @ W^T (+ bias) for any M, xq the activations rounded to e4m3 per token and block of 128
    (quantize_tokens_fp8): fp32 sums, one rounding to out_dtype.  The products are not exact: of 8 neighbouring k the f8
    matrix instruction drops what lies below 2^(e - 13), e the largest exponent sum among them, which was 1.5e-5 to 3.6e-5
    of a result on normal values (about 15 bits, with fp32 output too).  Arguments as fp8_w8a16_mm."""
    return _product(x, w, w_scale, bias, out_dtype, out_features, False)


def fp8_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
               out_features: Optional[int] = None) -> torch.Tensor:
    """A block-scaled FP8 linear layer: x bf16 [..., K] -> bf16 [..., N], fp8_w8a16_mm up to 16 rows and fp8_w8a8_mm above.
    ``torch.ops.qwen_fastpath.qf_fp8_linear`` is the same call as one opaque op for torch.compile."""
    if x.dim() == 2:
        return _product(x, w, w_scale, bias, _BF16, out_features, None)
    y = _product(x.reshape(-1, x.shape[-1]), w, w_scale, bias, _BF16, out_features, None)
    return y.view(*x.shape[:-1], y.shape[1])


@torch.library.custom_op("qwen_fastpath::qf_fp8_linear", mutates_args=(), device_types="cuda")
def qf_fp8_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  out_features: Optional[int] = None) -> torch.Tensor:
    return fp8_linear(x, w, w_scale, bias, out_features)


@qf_fp8_linear.register_fake
def _qf_fp8_linear_fake(x, w, w_scale, bias=None, out_features=None):
    N = w.shape[1] if w.dim() == 2 else w.numel() // x.shape[-1] if out_features is None else out_features
    return x.new_empty((*x.shape[:-1], N))
