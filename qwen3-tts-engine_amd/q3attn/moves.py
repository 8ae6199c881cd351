"""Moves of what a paged K/V pool holds, as torch ops over the q3attn C ABI: pages to other pages, and the kept tokens of rows to the
front of their pages, in all layers' caches in one launch.

Registered and behaving as the 8-bit pool's ops are (q3attn/fp8.py): GPU only, on the current stream, capturable, and in-place
operations on the caches.  The reference has neither: its seats own fixed pages and only grow (engine/talker.py:23-31, 42).
"""
from __future__ import annotations

from typing import Sequence

import torch

from ._lib import torch_op

_copy = torch_op("paged_copy", lambda caches, src, dst: None)
_compact = torch_op("paged_compact", lambda caches, keep, cache_seqlens, block_table, scales: torch.empty_like(cache_seqlens))


def paged_copy(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Page ``dst[i]`` of every cache becomes what its page ``src[i]`` is: ``cache[dst] = cache[src]`` for the whole list in one launch
    (of up to 128 caches of up to 4 shapes, in any order).  ``caches``: tensors [num_pages, ...] of any type, the pools of all layers, K and V, with
    their scales where they have some; src, dst [pairs] int32 on their device, as ``PagePool.fork``, ``unshare`` and ``defragment``
    return them.

    A page has to be made of runs of memory in at most two dimensions (a head-major view, some of the heads), addresses, runs and
    strides multiples of 4 bytes (of 16 in all caches: faster), and a call copies less than 8 GiB in a cache.

    Pages outside a cache (-1) are left out.  A page may be the source of several pairs; one that is the destination of two, or of one
    and another's source, holds a mix afterwards."""
    _copy(caches, src, dst)


def paged_compact(caches: Sequence[torch.Tensor], keep: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                  scales: Sequence[torch.Tensor] = ()) -> torch.Tensor:
    """Moves the kept tokens of each row to the front of its pages, in order and in place, and returns how many they are, [B] int32: the
    row's new cache_seqlens.  Token t < cache_seqlens[b] of row b is kept if ``keep[b, t]`` (bool [B, T]) is true, or if t >= T.  For
    long streams that let go of tokens, and for drafted tokens that were written and then rejected.  Keys stay as they are: a token
    keeps the rotary position that it was written with.

    ``caches``: the pools of all layers, K and V, bf16, 8-bit or 4-bit ([num_pages, page_size, Hkv, 128 or 64]), all of one shape and
    strides; ``scales``: their scales in the same order (``fp8_cache``, ``fp4_cache``; none for bf16).  ``block_table`` [B, max_pages]
    int32.  Rows with cache_seqlens <= 0 are left alone, and their cache_seqlens returned.  What lies behind the last kept token stays as
    it was.  Tokens whose page, or whose new place's page, the table does not give are not moved (but counted).  A row's pages from its
    first dropped token on must be its own: unshare forked ones first (``PagePool.unshare``); afterwards ``PagePool.truncate`` frees
    the pages behind."""
    return _compact(caches, keep, cache_seqlens, block_table, scales)
