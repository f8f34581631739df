"""A paged cache of keys and values in 4 bits, and attention over it, on MI355X.

The cache holds blocks of 32 values of a head that share a power of two, each value one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}
times it (e2m1): 17 bytes for 32 values, 0.27 of bf16.  Its records of 16 positions are laid out for the matrix
instructions' operands (include/qf_kv4.h).  ``qk_norm_rope`` and ``kv4_store`` write it, ``kv4_attention`` attends it (decode,
speculative verification, prompt chunks), ``kv4_load`` reads values back.  The kernels are hand-written HIP for gfx950; calls run
on torch's current stream of the tensors' device and may be captured in a HIP graph.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _kv4_lib as K
from .rope import _run


def kv4_cache(num_blocks: int, page_size: int, num_kv_heads: int, head_size: int, device="cuda") -> torch.Tensor:
    """An empty cache: uint8 [num_blocks, num_kv_heads, page_size / 16, 17 * head_size], zeros.  page_size a multiple of 16,
    head_size 64, 128 or 256.  Blocks may stand apart (a slice of a larger tensor's second dimension, as [:, layer])."""
    if head_size not in K.HEAD_SIZES or page_size < K.TILE or page_size % K.TILE or num_blocks < 1 or num_kv_heads < 1:
        raise ValueError(f"pages are multiples of {K.TILE}, head sizes {K.HEAD_SIZES}, got {page_size} and {head_size}")
    return torch.zeros(num_blocks, num_kv_heads, page_size // K.TILE, 17 * head_size, dtype=torch.uint8, device=device)


def kv4_store(key: torch.Tensor, value: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor) -> None:
    """key and value bf16 [T, H_kv, D] into the cache's slots (int64 [T]; those outside the cache, as -1, are not written; no
    two tokens may have one slot: their bytes could mix in it)."""
    if key.is_cuda:
        if K.try_call("rope", None, key, value, None, None, None, None, cache, slots, 0.0, 0.0, False, None, None) is not None:
            return
    K.head_size(key, "key")
    _run(None, key, None, None, None, None, value, cache, slots, 0.0, 0.0, False, None, None)


def kv4_load(cache: torch.Tensor, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(key, value) bf16 [T, H_kv, D]: what the cache holds at the slots (int64 [T]), exactly; zeros for slots outside it."""
    if cache.is_cuda:
        r = K.try_call("load", cache, slots)
        if r is not None:
            return r
    h, d, _ = K.cache_sizes(cache)
    dev = K.gpu(cache, slots)
    if slots.dim() != 1:
        raise TypeError(f"slots must be int64 [tokens], got {slots.dtype} {list(slots.shape)}")
    slots = K.vector(slots, torch.int64, slots.shape[0], "slots")
    if slots.shape[0] == 0:
        empty = cache.new_empty((0, h, d), dtype=torch.bfloat16)
        return empty, empty.clone()
    return K.call("load", dev, K.plain(cache), slots)


def kv4_attention(query: torch.Tensor, cache: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor, scale: float, *,
                  q_len: Optional[int] = None, cu_q: Optional[torch.Tensor] = None, max_q: Optional[int] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each request's new tokens over its cached positions (this step's among them):

        out[t, h] = sum_j softmax_j(scale * query[t, h] . key[j, h // G]) * value[j, h // G],    G = H // H_kv

    token i of the n of request b sees the positions j <= seq_lens[b] - n + i; a token that sees none gets zeros.  query bf16
    [T, H, D]; cache as kv4_cache's; seq_lens int32 [B]; block_table int32 [>= B, most pages].  Either q_len: every request has
    q_len tokens (token b * q_len + i), or cu_q int32 [B + 1], the first token of each request (StepTables.cu_q), with
    max_q, the most tokens a request may have.  Rows behind the last request's tokens are not written (out: as they were).
    out may be query itself.  At most 65535 requests.
    Lengths are kept inside the tables and block ids inside the cache.  Sums and the softmax are fp32; its weights are
    rounded to bf16 before they multiply the values, the output once."""
    if (q_len is None) == (cu_q is None) or (cu_q is None) != (max_q is None):
        raise ValueError("q_len is given, or cu_q with max_q")
    most = int(q_len if cu_q is None else max_q)
    if query.is_cuda:
        r = K.try_call("attention", query, cache, seq_lens, block_table, scale, most, cu_q, out)
        if r is not None:
            return r
    D = K.head_size(query, "query")
    T, H = query.shape[:2]
    h, d, page = K.cache_sizes(cache)
    dev = K.gpu(query, cache, seq_lens, block_table, cu_q, out)
    if d != D or H % h:
        raise ValueError(f"the cache holds {h} heads of {d} values, query has {H} of {D}")
    if seq_lens.dim() != 1:
        raise TypeError(f"seq_lens must be int32 [requests], got {seq_lens.dtype} {list(seq_lens.shape)}")
    B = seq_lens.shape[0]
    seq_lens = K.vector(seq_lens, torch.int32, B, "seq_lens")
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or block_table.shape[0] < B or block_table.shape[1] < 1:
        raise TypeError(f"block_table must be int32 [{B}, most pages], got {block_table.dtype} {list(block_table.shape)}")
    if (block_table.shape[1] > 1 and block_table.stride(1) != 1) or (
            block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]):
        block_table = block_table.contiguous()
    if block_table.shape[1] * page > 0x7FFFFFC0:
        raise ValueError(f"a row of the table holds up to {0x7FFFFFC0} positions, got {block_table.shape[1]} pages of {page}")
    if scale != scale:
        raise ValueError("scale is NaN")
    if most < 1:
        raise ValueError(f"a request has at least one token, got {most}")
    if cu_q is None:
        if B * most > T:
            raise ValueError(f"{B} requests of {most} tokens need {B * most} rows, query has {T}")
    else:
        cu_q = K.vector(cu_q, torch.int32, B + 1, "cu_q")
    out = K.output(out, (T, H, D), "out")
    query = K.heads(query, (T, H, D), "query")
    if T == 0 or B == 0:
        return query.new_empty((T, H, D)) if out is None else out
    return K.call("attention", dev, query, K.plain(cache), seq_lens, K.plain(block_table), scale, most, cu_q, out)
