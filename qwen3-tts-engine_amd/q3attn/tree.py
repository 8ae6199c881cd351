"""Attention for trees of drafted tokens over the paged K/V pool, as a torch custom op over the q3attn C ABI.

Speculative decoding checks several candidate continuations of a row in one pass: N drafted tokens, each of which sees the
row's cached tokens and its own ancestors in the tree of drafts.  GPU only.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import check, lib
from .fp8 import check_pool, check_rows, workspace
from .ops import _req, _stream


@torch.library.custom_op("q3attn::paged_decode_tree", mutates_args=())
def paged_decode_tree(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tree_mask: Optional[torch.Tensor],
                      k_cache: torch.Tensor, v_cache: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                      softmax_scale: float, k_scale: Optional[torch.Tensor] = None,
                      v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of N drafted tokens a row, q [B, N, Hq, 128] bf16 with k, v [B, N, Hkv, 128] bf16 (not in the pool; N <= 256):
    node n of row b sees the row's first cache_seqlens[b] cached tokens, gathered through ``block_table``, and node j's k, v if
    ``tree_mask`` (bool [B, N, N], or [N, N] for all rows) is true at [b, n, j]; None is a chain (j <= n).  The pool is bf16
    [num_pages, page_size, Hkv, 128], or 8-bit with ``k_scale``/``v_scale`` (``fp8_cache``).  Returns [B, N, Hq, 128] bf16.

    Rows with cache_seqlens < 0 are skipped and give zeros, as does a node that sees nothing.  Rows with fewer drafts pad N and
    leave the padding out of the mask: what padded (masked) k and v rows hold does not matter.  Only ``out`` is written; the
    accepted nodes' k and v go into the pool afterwards (``paged_write_fp8`` with slot -1 for the rejected, or an index_copy_
    for the bf16 pool).  The reference decodes one token a row (engine/talker.py:77); with N = 1 and no mask this is its call
    with the new token not yet in the cache."""
    who = "q3attn.paged_decode_tree"
    _req(q.is_cuda, f"{who}: tensors must be on a GPU (there is no CPU path)")
    dev = q.device
    _req(q.dim() == 4 and k.dim() == 4 and v.dim() == 4 and k_cache.dim() == 4,
         f"{who}: q, k, v must be [batch, nodes, heads, head_dim] and the caches [num_pages, page_size, kv_heads, head_dim]")
    B, N, Hq, D = q.shape
    pages, page, Hkv, Dc = k_cache.shape
    for name, t, shape in (("q", q, (B, N, Hq, Dc)), ("k", k, (B, N, Hkv, Dc)), ("v", v, (B, N, Hkv, Dc))):
        _req(t.device == dev and t.dtype == torch.bfloat16, f"{who}: {name} must be bfloat16 on {dev}")
        _req(t.shape == shape and t.stride(3) == 1, f"{who}: {name} must be {shape} with a contiguous head_dim")
    _req((k_scale is None) == (v_scale is None), f"{who}: pass both k_scale and v_scale, or neither")
    if k_scale is not None:
        check_pool(who, dev, k_cache, v_cache, k_scale, v_scale)
        scales = (k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), k_scale.stride(1))
    else:
        _req(k_cache.device == dev and v_cache.device == dev and k_cache.dtype == torch.bfloat16
             and v_cache.dtype == torch.bfloat16, f"{who}: without scales k_cache/v_cache must be bfloat16 on {dev}")
        _req(k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride() and k_cache.stride(3) == 1,
             f"{who}: k_cache and v_cache must have the same shape and strides, dim contiguous")
        scales = (None, None, 0, 0)
    check_rows(who, dev, B, cache_seqlens, block_table)
    mask = (None, 0, 0)
    if tree_mask is not None:
        _req(tree_mask.device == dev and tree_mask.dtype == torch.bool, f"{who}: tree_mask must be bool on {dev}")
        _req(tree_mask.shape == (B, N, N) or tree_mask.shape == (N, N), f"{who}: tree_mask must be [{B}, {N}, {N}] or [{N}, {N}]")
        _req(tree_mask.stride(-1) == 1 or N <= 1, f"{who}: tree_mask rows must be contiguous")
        mask = (tree_mask.data_ptr(), tree_mask.stride(0) if tree_mask.dim() == 3 else 0, tree_mask.stride(-2))
    out = torch.empty((B, N, Hq, D), dtype=q.dtype, device=dev)
    if B == 0 or N == 0:
        return out
    L = lib()
    with torch.cuda.device(dev):
        ws, nbytes = workspace(L, B, N, Hq, Hkv, D, block_table.shape[1], page, dev)
        rc = L.q3a_paged_decode_tree(
            q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), k.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
            v.data_ptr(), v.stride(0), v.stride(1), v.stride(2), *mask,
            k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), *scales,
            pages, page, cache_seqlens.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            out.data_ptr(), out.stride(0), out.stride(1), out.stride(2), ws.data_ptr() if ws is not None else None, nbytes,
            B, N, Hq, Hkv, D, float(softmax_scale), _stream(dev))
    check(rc, "q3a_paged_decode_tree")
    return out


@paged_decode_tree.register_fake
def _paged_decode_tree_fake(q, k, v, tree_mask, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, k_scale=None,
                            v_scale=None):
    return torch.empty_like(q, memory_format=torch.contiguous_format)
