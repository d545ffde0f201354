"""Block tables and slots of a serving step, made on the GPU: what stands in front of the prologue, which takes slots and positions, and of the
attention, which takes block tables, lengths and starts.

Request r has `context_lens[r]` tokens in the paged cache and gets `new_lens[r]` more (a chunk of its prompt, one token, or none; negative
numbers count as none).  Entry i of its row of `block_table` is the cache block of its tokens i * cache_block_size on.

* `extend_block_tables` takes the blocks that the new tokens need from a stack of free ones and lists the step's tokens.
* `release_block_tables` puts the blocks of finished requests back onto the stack.

Both only read numbers that are on the GPU, so a step can be captured in a graph with its lengths and its pool as state: `out.seq_lens` may be
`context_lens` itself, and the `num_free` of a result `num_free` itself.  No other result may share memory with another argument: the library
refuses that (`Dsv4Error`).  Calls on one pool have to follow one another.  A count of free blocks below zero counts as none, one above the
stack's capacity as all of it.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch

from .. import _native

MOST_REQUESTS = 8192


class PagedBatch(NamedTuple):
    """The tokens of a step, request by request."""

    query_start_loc: torch.Tensor  # int32 [requests + 1]: sums of the new lengths
    seq_lens: torch.Tensor  # int32 [requests]: context and new tokens
    position_ids: torch.Tensor  # int64 [num_tokens]
    slot_mapping: torch.Tensor  # int64 [num_tokens]; -1: not cached
    token_to_req_indices: torch.Tensor  # int32 [num_tokens]
    num_free: torch.Tensor  # int32 [1]: blocks that are left on the stack
    num_missing: torch.Tensor  # int32 [1]: blocks that were not there


_extend = _release = None  # the native front ends, looked up once


def _bind():
    global _extend, _release
    calls = _native.host_calls()
    _extend, _release = calls.extend_block_tables, calls.release_block_tables


def extend_block_tables(
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_blocks: torch.Tensor,
    num_free: torch.Tensor,
    cache_block_size: int,
    num_tokens: int,
    out: Optional[Sequence[torch.Tensor]] = None,
) -> PagedBatch:
    """Fills the entries of `block_table` that the new tokens need and returns the step's `PagedBatch` (in the tensors of `out`, where given).

    The first num_free[0] entries of `free_blocks` are a stack whose last one is taken first, in the order of requests and of their entries; the
    stack itself is not written, what is left of it is the result's `num_free`.  Where it is empty the entry becomes -1, the tokens in it get
    the slot -1, and `num_missing` counts the entry: the caller has to take such a batch back or release other requests.  Entries behind the table's
    width have no place: no block is taken, and the tokens get the slot -1.

    `num_tokens` is the length of the per-token results: the tokens beyond it are left out, and rows behind the last token (a batch that is
    padded to a captured size) have the slot -1, position 0 and request 0.

    Args:
        context_lens, new_lens: [requests <= 8192] int32
        block_table: [requests, blocks] int32 with unit inner stride, modified in place
        free_blocks: [capacity] int32, read only
        num_free: [1] int32
        cache_block_size: tokens per cache block
        num_tokens: rows of the per-token results
        out: the seven tensors of a PagedBatch; none may share memory with another argument, but seq_lens may be context_lens and
            num_free the argument of that name
    """
    if _extend is None:
        _bind()
    result = _extend(context_lens, new_lens, block_table, free_blocks, num_free, cache_block_size, num_tokens, *(out or ()))
    if result is True:
        return out if isinstance(out, PagedBatch) else PagedBatch._make(out)
    if result is not None:
        return PagedBatch._make(result)
    _check_pool(context_lens, block_table, free_blocks, num_free, cache_block_size)
    requests, num_tokens = context_lens.shape[0], int(num_tokens)
    _check_list("new_lens", new_lens, torch.int32, requests, context_lens)
    assert 0 <= num_tokens < 1 << 31
    if out:
        assert len(out) == len(PagedBatch._fields), "out: the seven tensors of a PagedBatch"
        sizes = (requests + 1, requests, num_tokens, num_tokens, num_tokens, 1, 1)
        for i, (name, t, size) in enumerate(zip(PagedBatch._fields, out, sizes)):
            _check_list(name, t, torch.int64 if i in (2, 3) else torch.int32, size, context_lens)
    _native.refuse()


def release_block_tables(
    seq_lens: torch.Tensor,
    finished: torch.Tensor,
    block_table: torch.Tensor,
    free_blocks: torch.Tensor,
    num_free: torch.Tensor,
    cache_block_size: int,
    num_free_out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Puts the blocks of the requests with `finished` onto the stack `free_blocks`, as many as their `seq_lens` tokens take, the last one first:
    what undoes `extend_block_tables`.  Negative entries (blocks that were missing) are left out.  Returns how many the stack has now, in
    `num_free_out` where given (which may be `num_free`).

    `block_table` stays as it is; the next request of the row starts with a context of 0.  A request is released once: a second time would put its
    blocks on the stack twice.  `free_blocks` has to have a place for every block of the cache; blocks beyond its end are dropped.

    Args:
        seq_lens: [requests <= 8192] int32
        finished: [requests] bool
        block_table: [requests, blocks] int32 with unit inner stride, read only
        free_blocks: [capacity] int32, modified in place from entry num_free[0] on
        num_free, num_free_out: [1] int32
        cache_block_size: tokens per cache block
    """
    if _release is None:
        _bind()
    result = _release(seq_lens, finished, block_table, free_blocks, num_free, cache_block_size, num_free_out)
    if result is not None:
        return result
    _check_pool(seq_lens, block_table, free_blocks, num_free, cache_block_size)
    _check_list("finished", finished, torch.bool, seq_lens.shape[0], seq_lens)
    if num_free_out is not None:
        _check_list("num_free_out", num_free_out, torch.int32, 1, seq_lens)
    _native.refuse()


def _check_list(name, t, dtype, size, first):
    assert t.dim() == 1 and t.dtype == dtype and t.shape[0] == size and t.is_contiguous(), f"{name}: {dtype} [{size}], contiguous"
    assert t.device == first.device, "all tensors must be on the same device"


def _check_pool(lens, block_table, free_blocks, num_free, cache_block_size):
    assert lens.device.type == "cuda", "this operator has no CPU path"
    assert lens.dim() == 1 and lens.dtype == torch.int32 and lens.is_contiguous(), "lengths: int32 [requests], contiguous"
    assert lens.shape[0] <= MOST_REQUESTS, f"at most {MOST_REQUESTS} requests"
    assert 0 < int(cache_block_size) < 1 << 31
    assert block_table.dim() == 2 and block_table.dtype == torch.int32 and block_table.stride(1) == 1, "block_table: int32 [requests, blocks] with unit inner stride"
    assert block_table.shape[0] == lens.shape[0], "a row of block_table per request"
    assert block_table.shape[0] <= 1 or block_table.stride(0) >= block_table.shape[1], "rows of block_table must not overlap"
    assert free_blocks.dim() == 1 and free_blocks.dtype == torch.int32 and free_blocks.is_contiguous(), "free_blocks: int32 [capacity], contiguous"
    assert block_table.numel() < 1 << 31 and free_blocks.numel() < 1 << 31
    for t in (block_table, free_blocks):
        assert t.device == lens.device, "all tensors must be on the same device"
    _check_list("num_free", num_free, torch.int32, 1, lens)


__all__ = ["PagedBatch", "extend_block_tables", "release_block_tables"]
