"""Attention for trees of drafted tokens over the paged K/V pool, as a torch op over the q3attn C ABI.

Speculative decoding checks several candidate continuations of a row in one pass: N drafted tokens, each of which sees the
row's cached tokens and its own ancestors in the tree of drafts.  Registered from C++ as the 8-bit pool's ops are.  GPU only.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import torch_op

_tree = torch_op("paged_decode_tree", lambda q, *rest, **more: torch.empty_like(q, memory_format=torch.contiguous_format))


def paged_decode_tree(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tree_mask: Optional[torch.Tensor],
                      k_cache: torch.Tensor, v_cache: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                      softmax_scale: float, k_scale: Optional[torch.Tensor] = None,
                      v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of N drafted tokens a row, q [B, N, Hq, 128] bf16 with k, v [B, N, Hkv, 128] bf16 (not in the pool; N <= 256):
    node n of row b sees the row's first cache_seqlens[b] cached tokens, gathered through ``block_table``, and node j's k, v if
    ``tree_mask`` (bool [B, N, N], or [N, N] for all rows) is true at [b, n, j]; None is a chain (j <= n).  The pool is bf16
    [num_pages, page_size, Hkv, 128], or 8-bit with ``k_scale``/``v_scale`` (``fp8_cache``).  Returns [B, N, Hq, 128] bf16.

    Rows with cache_seqlens < 0 are skipped and give zeros, as does a node that sees nothing.  Rows with fewer drafts pad N and
    leave the padding out of the mask: what padded (masked) k and v rows hold does not matter.  Only the result is written; the
    accepted nodes' k and v go into the pool afterwards (``paged_write_fp8`` with slot -1 for the rejected, or an index_copy_
    for the bf16 pool).  The reference decodes one token a row (engine/talker.py:77); with N = 1 and no mask this is its call
    with the new token not yet in the cache."""
    return _tree(q, k, v, tree_mask, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, k_scale, v_scale)
