"""Block tables and slot maps of a batch of requests, built on the GPU from their lengths.

The reference cache is dense (entmaxkv/kv_cache.py:44-56) and has no counterpart.  ``PagedKVCache`` with
``num_blocks`` calls both functions for its own pool; a serving engine that owns its pool calls them itself.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib

#: sequences per call
MAX_BATCH = 16384


def _check(seq_lens, other, block_table, free_blocks, page_size, name, *outputs):
    """(B, device index, other is a tensor) of arguments that hold together."""
    per_row = isinstance(other, torch.Tensor)
    index = _lib.require_on_one_device(seq_lens, other if per_row else None, block_table, free_blocks, *outputs)
    shape, table = seq_lens.shape, block_table.shape
    if seq_lens.dtype != torch.int32 or len(shape) != 1 or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous int32 [B] tensor")
    B = shape[0]
    if B > MAX_BATCH:
        raise ValueError(f"at most {MAX_BATCH} sequences per call")
    if per_row:
        if other.dtype != torch.int32 or other.shape != shape or not other.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 [B] tensor or an int")
    elif isinstance(other, bool) or not isinstance(other, int) or not 0 <= other < 1 << 31:
        raise ValueError(f"{name} must be a contiguous int32 [B] tensor or an int >= 0")
    if block_table.dtype != torch.int32 or len(table) != 2 or table[0] != B or (
            not block_table.is_contiguous() and ((table[1] > 1 and block_table.stride(1) != 1)
                                                 or (B > 1 and block_table.stride(0) < table[1]))):
        raise ValueError("block_table must be int32 [B, pages], contiguous along the pages")
    if free_blocks.dtype != torch.int32 or free_blocks.dim() != 1 or not free_blocks.is_contiguous():
        raise ValueError("free_blocks must be a contiguous int32 [num_blocks] tensor")
    if page_size <= 0:
        raise ValueError("page_size must be positive")
    return B, index, per_row


def plan_block_tables(seq_lens: torch.Tensor, new_lens: Union[torch.Tensor, int], block_table: torch.Tensor,
                      free_blocks: torch.Tensor, page_size: int, slots: Optional[torch.Tensor] = None,
                      positions: Optional[torch.Tensor] = None, row_starts: Optional[torch.Tensor] = None,
                      status: Optional[torch.Tensor] = None):
    """Give the pages that ``new_lens[b]`` more tokens of every sequence need their blocks, and the tokens their slots.

    seq_lens int32 [B]: tokens that each sequence holds, on ``ceil(seq_lens / page_size)`` pages; new_lens int32 [B] or
    one int for all.  ``free_blocks`` int32 [num_blocks] is the pool as a stack: its lowest ``sum(held pages)`` places
    are in use (their content does not matter), and the missing pages take the places from there on in sequence order,
    -1 once the pool is used up.  A sequence gets no pages behind the table's width.  ``block_table`` int32 [B, pages]
    gets those entries and keeps the others.

    The new tokens of all sequences one after another get ``slots`` (int64: block * page_size + place in the page, -1
    without a block) and ``positions`` (int32), both -1 behind the last token; ``row_starts`` (int32 [B + 1]) says where
    each sequence's tokens begin.  Lengths are not changed: the call can be repeated, and what it planned is in use once
    ``seq_lens`` has grown.  ``status`` (int32, optional) gets bit 2 (capacity) when the pool or the table did not
    suffice.  Returns (block_table, slots, positions, row_starts).
    """
    B, index, per_row = _check(seq_lens, new_lens, block_table, free_blocks, page_size, "new_lens", slots, positions,
                               row_starts, status)
    n = 0
    if slots is not None:
        n = slots.shape[0] if slots.dim() == 1 else -1
        if slots.dtype != torch.int64 or n < 0 or not slots.is_contiguous():
            raise ValueError("slots must be contiguous int64, one entry per token")
    if positions is not None:
        m = positions.shape[0] if positions.dim() == 1 else -1
        if positions.dtype != torch.int32 or m < 0 or not positions.is_contiguous() or (slots is not None and m != n):
            raise ValueError("positions must be contiguous int32, one entry per token, as many as slots")
        n = m
    if row_starts is not None and (row_starts.dtype != torch.int32 or row_starts.shape != (B + 1,)
                                   or not row_starts.is_contiguous()):
        raise ValueError("row_starts must be a contiguous int32 [B + 1] tensor")
    if status is not None and status.dtype != torch.int32:
        raise ValueError("status must be int32")
    width = block_table.shape[1]
    with _lib.on_device(index):
        _lib.check(_lib.load().ekv_plan_block_tables(
            seq_lens.data_ptr(), new_lens.data_ptr() if per_row else None, 0 if per_row else new_lens, B, page_size,
            block_table.data_ptr(), block_table.stride(0) if B > 1 else width, width, free_blocks.data_ptr(),
            free_blocks.shape[0], _lib.ptr(slots), _lib.ptr(positions), n, _lib.ptr(row_starts), _lib.ptr(status),
            _lib.stream_ptr()), "ekv_plan_block_tables")
    return block_table, slots, positions, row_starts


def release_block_tables(seq_lens: torch.Tensor, keep_lens: Union[torch.Tensor, int], block_table: torch.Tensor,
                         free_blocks: torch.Tensor, page_size: int, status: Optional[torch.Tensor] = None):
    """Return the pages behind the first ``keep_lens[b]`` tokens of every sequence to ``free_blocks`` and lower
    ``seq_lens`` to ``keep_lens`` (arguments as ``plan_block_tables``); their table entries become -1."""
    return_blocks(seq_lens, keep_lens, block_table, free_blocks, page_size, status)
    with _lib.on_device(seq_lens.get_device()):
        if isinstance(keep_lens, torch.Tensor):
            torch.minimum(seq_lens, keep_lens.clamp(min=0), out=seq_lens)
        else:
            seq_lens.clamp_(max=keep_lens)
    return block_table


def return_blocks(seq_lens, keep_lens, block_table, free_blocks, page_size, status=None) -> None:
    """``release_block_tables`` without lowering the lengths."""
    B, index, per_row = _check(seq_lens, keep_lens, block_table, free_blocks, page_size, "keep_lens", status)
    if status is not None and status.dtype != torch.int32:
        raise ValueError("status must be int32")
    width = block_table.shape[1]
    with _lib.on_device(index):
        _lib.check(_lib.load().ekv_release_blocks(
            seq_lens.data_ptr(), keep_lens.data_ptr() if per_row else None, 0 if per_row else keep_lens, B, page_size,
            block_table.data_ptr(), block_table.stride(0) if B > 1 else width, width, free_blocks.data_ptr(),
            free_blocks.shape[0], _lib.ptr(status), _lib.stream_ptr()), "ekv_release_blocks")
