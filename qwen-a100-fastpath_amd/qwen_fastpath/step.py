"""A step's tables, built on the GPU from request lengths.

Between two steps of a serving loop the requests' lengths change (accepted draft tokens, prompt chunks), and what the kernels
read follows from them: each token's position and cache slot, the block table with the pages newly taken, the lengths.
``step_tables`` makes all of it in one launch (qf_step_tables, include/qf_kv4.h), so that a loop whose lengths stand on the GPU
need not bring them to the host, and a whole step may be captured in a HIP graph.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _kv4_lib as K

_I32 = torch.int32


class StepTables(NamedTuple):
    """Tokens stand one after the other, request after request."""
    cu_q: torch.Tensor        # int32 [requests + 1]: the first token of each request, then their number
    seq_lens: torch.Tensor    # int32 [requests]: cached positions, this step's tokens included
    positions: torch.Tensor   # int64 [tokens]: of each token in its request; 0 behind the last
    slots: torch.Tensor       # int64 [tokens]: block * page size + place; -1 behind the last
    held: torch.Tensor        # int32 [requests]: pages each request holds now
    free_count: torch.Tensor  # int32 [1]: blocks left on the stack
    fits: torch.Tensor        # int32 [1]: 1; 0 where the step did not fit and nothing was taken


def step_tables(context_lens: torch.Tensor, query_lens: torch.Tensor, held: torch.Tensor, block_table: torch.Tensor,
                free_blocks: torch.Tensor, free_count: torch.Tensor, page_size: int, num_tokens: int) -> StepTables:
    """The tables of a step in which request b, with context_lens[b] cached positions and held[b] pages (the first entries of its
    row of block_table int32 [requests, most pages]), gets query_lens[b] new tokens.

    The pages it lacks are taken from the top of the stack free_blocks[: free_count] (request after request; the last block
    first) and entered into block_table in place; the stack itself stays as it is, the returned count says what is left of it.
    num_tokens: the length of positions and slots, at least the tokens of the step (the size a captured step is padded to).
    A step that does not fit (too many tokens, pages or blocks, a negative length) takes nothing: fits is 0, every slot -1,
    cu_q all 0, the lengths the contexts'.  Lengths and counts are int32 on the GPU; at most 4096 requests."""
    if context_lens.is_cuda:
        r = K.try_call("tables", context_lens, query_lens, held, block_table, free_blocks, free_count, int(page_size), int(num_tokens))
        if r is not None:
            return StepTables(*r)
    if context_lens.dim() != 1 or not 1 <= context_lens.shape[0] <= K.MAX_REQS:
        raise ValueError(f"context_lens must be [1..{K.MAX_REQS}], got {list(context_lens.shape)}")
    dev = K.gpu(context_lens, query_lens, held, block_table, free_blocks, free_count)
    B, page_size, num_tokens = context_lens.shape[0], int(page_size), int(num_tokens)
    context_lens, query_lens, held = (K.vector(t, _I32, B, n) for t, n in (
        (context_lens, "context_lens"), (query_lens, "query_lens"), (held, "held")))
    free_count = K.vector(free_count, _I32, 1, "free_count")
    if free_blocks.dim() != 1 or free_blocks.shape[0] > K.MAX_TOKENS:
        raise ValueError(f"free_blocks must be one row of at most {K.MAX_TOKENS} blocks, got {list(free_blocks.shape)}")
    free_blocks = K.vector(free_blocks, _I32, free_blocks.shape[0], "free_blocks")
    if block_table.dtype is not _I32 or block_table.dim() != 2 or block_table.shape[0] < B or not (
            1 <= block_table.shape[1] <= K.MAX_TOKENS):
        raise TypeError(f"block_table must be int32 [{B}, most pages], got {block_table.dtype} {list(block_table.shape)}")
    if (block_table.shape[1] > 1 and block_table.stride(1) != 1) or (
            block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError(f"block_table must have rows that are contiguous and apart, got strides {block_table.stride()}")
    if not 1 <= page_size <= 0x7FFFFFFF:
        raise ValueError(f"page_size must be positive, got {page_size}")
    if not 0 <= num_tokens <= K.MAX_TOKENS:
        raise ValueError(f"num_tokens must be in [0, {K.MAX_TOKENS}], got {num_tokens}")
    return StepTables(*K.call("tables", dev, context_lens, query_lens, held, K.plain(block_table), free_blocks, free_count, page_size,
                              num_tokens))
