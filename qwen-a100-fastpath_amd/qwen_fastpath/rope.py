"""Norms of the query and key heads with the position rotation and the write into the cache, on MI355X.

Between a layer's qkv product and its attention stand a norm of each query and key head, the rotation of its first values by
the token's position, and the write of keys and values into the paged cache; ``qk_norm_rope`` does all of it in one launch
and one pass over the data (qf_qk_norm_rope, include/qf_kv4.h), for the bf16 pages that ``gqa_packed_spec_attention`` reads and
for the 4-bit cache of ``kv4_attention``.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _kv4_lib as K

_BF16 = torch.bfloat16


def qk_norm_rope(query: torch.Tensor, key: torch.Tensor, positions: Optional[torch.Tensor], cos_sin: Optional[torch.Tensor],
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
                 value: Optional[torch.Tensor] = None,
                 cache: Union[None, torch.Tensor, Tuple[torch.Tensor, torch.Tensor]] = None,
                 slots: Optional[torch.Tensor] = None, eps: float = 1e-6, weight_offset: float = 0.0, interleaved: bool = False,
                 query_out: Optional[torch.Tensor] = None,
                 key_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(query, key) with each head normalised and turned:

        n = x * rsqrt(mean(x^2) + eps) * (weight_offset + weight)      (x itself where the weight is None)
        pairs (a, b) of the first rot values -> (a cos - b sin, b cos + a sin)

    query bf16 [T, H, D], key (and value) bf16 [T, H_kv, D], any strides that are multiples of 8 (views of a qkv product's
    output); weights bf16 [D] (weight_offset 1 for checkpoints that store them less one); cos_sin bf16 or fp32 [positions,
    rot]: each position's cosines, then its sines, rot a multiple of 16 up to D; positions int64 [T], kept inside the table; both
    None: no rotation.  A pair is (i, i + rot / 2), or (2 i, 2 i + 1) with `interleaved`.  D is 64, 128 or 256.

    With a cache, the key and the value go to the slots (int64 [T]; those outside the cache, as -1, are not written; no two
    tokens may have one slot: their bytes could mix in it).  `cache` is (key_cache, value_cache), bf16 [blocks, page, H_kv, D],
    or a 4-bit cache (kv4_cache).  The key is returned only where key_out is given, or without a cache.  query_out and key_out
    may be query and key (in place); no other overlap.
    Arithmetic is fp32 with one rounding to bf16; keys for the 4-bit cache are computed in fp64, rounded to bf16 and these
    values quantised, so that a token's codes do not depend on the order of a sum."""
    if key.is_cuda:
        r = K.try_call("rope", query, key, value, positions, cos_sin, q_weight, k_weight, cache, slots, eps, weight_offset,
                       interleaved, query_out, key_out)
        if r is not None:
            return r
    D = K.head_size(query, "query")
    if key.dim() != 3 or key.shape[0] != query.shape[0] or key.shape[2] != D or key.shape[1] < 1:
        raise ValueError(f"key must be [{query.shape[0]}, kv heads, {D}], got {list(key.shape)}")
    return _run(query, key, positions, cos_sin, q_weight, k_weight, value, cache, slots, eps, weight_offset, interleaved, query_out,
                key_out)


def _run(query, key, positions, cos_sin, q_weight, k_weight, value, cache, slots, eps, weight_offset, interleaved, query_out,
         key_out):
    """The call checked, with the copies that the kernels need.  query None: keys and values alone."""
    T, HK, D = key.shape
    pages = () if cache is None else tuple(cache) if isinstance(cache, (tuple, list)) else (cache,)
    dev = K.gpu(key, query, value, positions, cos_sin, q_weight, k_weight, slots, query_out, key_out, *pages)
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if query is not None:
        H = query.shape[1]
        query_out = K.output(query_out, (T, H, D), "query_out")
        query = K.heads(query, (T, H, D), "query")
    key_out = K.output(key_out, (T, HK, D), "key_out")
    key = K.heads(key, (T, HK, D), "key")
    q_weight, k_weight = (None if w is None else K.vector(w, _BF16, D, n, 16) for w, n in (
        (q_weight, "q_weight"), (k_weight, "k_weight")))
    if (cos_sin is None) != (positions is None):
        raise ValueError("positions and cos_sin are given together, or neither")
    if cos_sin is not None:
        if cos_sin.dtype not in (_BF16, torch.float32) or cos_sin.dim() != 2 or cos_sin.shape[0] < 1:
            raise TypeError(f"cos_sin must be bf16 or fp32 [positions, rot], got {cos_sin.dtype} {list(cos_sin.shape)}")
        if cos_sin.shape[1] % 16 or not 16 <= cos_sin.shape[1] <= D:
            raise ValueError(f"rot must be a multiple of 16 up to {D}, got {cos_sin.shape[1]}")
        if not cos_sin.is_contiguous() or cos_sin.data_ptr() % 16:
            cos_sin = cos_sin.clone(memory_format=torch.contiguous_format)
        cos_sin = K.plain(cos_sin)
        positions = K.vector(positions, torch.int64, T, "positions")
    if cache is None:
        if value is not None or slots is not None:
            raise ValueError("value and slots go with a cache")
    else:
        if value is None or slots is None:
            raise ValueError("a cache takes value and slots")
        value = K.heads(value, (T, HK, D), "value")
        slots = K.vector(slots, torch.int64, T, "slots")
        if len(pages) == 1:
            h, d, _ = K.cache_sizes(pages[0])
            if (h, d) != (HK, D):
                raise ValueError(f"the cache holds {h} heads of {d} values, key {HK} of {D}")
            cache = K.plain(pages[0])
        else:
            if len(pages) != 2:
                raise TypeError("cache is a 4-bit cache or (key_cache, value_cache)")
            for t, n in zip(pages, ("key_cache", "value_cache")):
                if t.dtype is not _BF16 or t.dim() != 4 or 0 in t.shape or tuple(t.shape[2:]) != (HK, D) or t.shape != pages[0].shape:
                    raise TypeError(f"{n} must be bf16 [blocks, page, {HK}, {D}] (both alike), got {t.dtype} {list(t.shape)}")
                if t.stride(3) != 1 or t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:3]):
                    raise ValueError(f"{n} must be 16-byte aligned, its last dimension contiguous and its strides multiples of 8, got "
                                     f"{t.stride()}")
                if K.overlaps(t):
                    raise ValueError(f"{n} is written, its heads must not share memory, got strides {t.stride()}")
            cache = tuple(K.plain(t) for t in pages)
    if T == 0:
        return (query_out if query is None or query_out is not None else torch.empty_like(query),
                key_out if cache is not None or key_out is not None else torch.empty_like(key))
    return K.call("rope", dev, query, key, value, positions, cos_sin, q_weight, k_weight, cache, slots, eps, weight_offset,
                  interleaved, query_out, key_out)
