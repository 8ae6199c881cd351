"""The 8-bit K/V pool as torch custom ops over the q3attn C ABI: its buffers, the quantising write, the read back, and decode
attention over it.

A pool row (one token of one KV head, 128 values) is held as e4m3 codes and one exponent byte s, value = code * 2^(s - 127):
the smallest power of two that takes the row's largest finite magnitude to at most 448 (at least 2^-117; elements that are not
finite are held as NaN).  A row takes 129 bytes instead of 256.  The scale being a power of two, every value read back is a bf16
number, and attention over the pool is attention over the bf16 rows that ``paged_read_fp8`` returns.  GPU only.
"""
from __future__ import annotations

import torch

from ._lib import check, lib
from .ops import _req, _stream

E4M3 = torch.float8_e4m3fn


def fp8_cache(num_pages: int, page_size: int = 16, num_kv_heads: int = 8, head_dim: int = 128, device="cuda"):
    """Buffers of one layer's 8-bit pool: (k_cache, v_cache, k_scale, v_scale), k/v_cache [num_pages, page_size, kv_heads,
    head_dim] float8_e4m3fn and k/v_scale [num_pages, kv_heads, page_size] uint8, all holding the value 0.  The caches are
    views whose memory holds a page's tokens of one head next to each other, so a head's page is one run of memory; the ops
    take any strides."""
    caches = [torch.zeros((num_pages, num_kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(E4M3)
              .transpose(1, 2) for _ in range(2)]
    scales = [torch.full((num_pages, num_kv_heads, page_size), 127, dtype=torch.uint8, device=device) for _ in range(2)]
    return (*caches, *scales)


def check_pool(who, dev, k_cache, v_cache, k_scale, v_scale):
    """The checks of an 8-bit pool on ``dev`` that the C entry points cannot make."""
    _req(k_cache.device == dev and v_cache.device == dev and k_scale.device == dev and v_scale.device == dev,
         f"{who}: the pool and its scales must be on {dev}")
    _req(k_cache.dtype == E4M3 and v_cache.dtype == E4M3, f"{who}: k_cache/v_cache must be float8_e4m3fn")
    _req(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride()
         and k_cache.stride(3) == 1,
         f"{who}: k_cache and v_cache must be [num_pages, page_size, kv_heads, head_dim] with equal strides")
    pages, page, Hkv, _ = k_cache.shape
    _req(k_scale.dtype == torch.uint8 and v_scale.dtype == torch.uint8, f"{who}: k_scale/v_scale must be uint8")
    _req(k_scale.shape == (pages, Hkv, page) and v_scale.shape == k_scale.shape and k_scale.stride() == v_scale.stride()
         and k_scale.stride(2) == 1,
         f"{who}: k_scale and v_scale must be [num_pages, kv_heads, page_size] with equal strides and contiguous tokens")


def check_rows(who, dev, B, cache_seqlens, block_table):
    _req(cache_seqlens.device == dev and block_table.device == dev,
         f"{who}: cache_seqlens and block_table must be on {dev}")
    _req(cache_seqlens.dtype == torch.int32 and cache_seqlens.shape == (B,) and cache_seqlens.is_contiguous(),
         f"{who}: cache_seqlens must be a contiguous int32 [batch] tensor")
    _req(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B
         and (block_table.stride(1) == 1 or block_table.shape[1] <= 1),
         f"{who}: block_table must be int32 [batch, max_pages] with contiguous rows")


def _tokens(who, x, name, dev):
    _req(x.device == dev, f"{who}: {name} is on {x.device}, the pool on {dev}")
    _req(x.dtype == torch.bfloat16 and x.dim() == 3 and x.stride(2) == 1,
         f"{who}: {name} must be bfloat16 [tokens, kv_heads, head_dim] with a contiguous head_dim")


def _slots(who, slots, dev):
    _req(slots.device == dev and slots.dtype == torch.int64 and slots.dim() == 1 and slots.is_contiguous(),
         f"{who}: slots must be a contiguous int64 [tokens] tensor on the pool's device")


@torch.library.custom_op("q3attn::paged_write_fp8", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def paged_write_fp8(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Quantise rows k, v [T, Hkv, 128] bf16 (any token and head strides) into the 8-bit pool: token t at ``slots[t]`` = page *
    page_size + offset (int64, as ``PagePool.slot`` gives them); a slot outside the pool (-1) is not written.  A slot given to
    two tokens holds a mix of both afterwards, so only a scratch slot that nothing reads may be given twice.  For this pool
    what the index_copy_ pair of engine/talker.py:72-73 and :161-162 is for the bf16 one."""
    who = "q3attn.paged_write_fp8"
    _req(k_cache.is_cuda, f"{who}: tensors must be on a GPU (there is no CPU path)")
    dev = k_cache.device
    check_pool(who, dev, k_cache, v_cache, k_scale, v_scale)
    _slots(who, slots, dev)
    _tokens(who, k, "k", dev)
    _tokens(who, v, "v", dev)
    pages, page, Hkv, D = k_cache.shape
    T = slots.shape[0]
    _req(k.shape == (T, Hkv, D) and v.shape == (T, Hkv, D), f"{who}: k and v must be [{T}, {Hkv}, {D}]")
    if T == 0:
        return
    with torch.cuda.device(dev):
        rc = lib().q3a_paged_write_fp8(
            k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), k_scale.stride(1), pages, page, T, Hkv, D, _stream(dev))
    check(rc, "q3a_paged_write_fp8")


@paged_write_fp8.register_fake
def _paged_write_fp8_fake(k, v, slots, k_cache, v_cache, k_scale, v_scale):
    return None


@torch.library.custom_op("q3attn::paged_read_fp8", mutates_args=())
def paged_read_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                   slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows of ``slots`` [T] int64 as (k, v) [T, Hkv, 128] bf16, exactly as the pool holds them: the packed K/V that
    ``flash_attn_varlen_func`` takes, for a prefill over a cached prefix.  Slots outside the pool (-1) read zeros."""
    who = "q3attn.paged_read_fp8"
    _req(k_cache.is_cuda, f"{who}: tensors must be on a GPU (there is no CPU path)")
    dev = k_cache.device
    check_pool(who, dev, k_cache, v_cache, k_scale, v_scale)
    _slots(who, slots, dev)
    pages, page, Hkv, D = k_cache.shape
    T = slots.shape[0]
    k = torch.empty((T, Hkv, D), dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    if T == 0:
        return k, v
    with torch.cuda.device(dev):
        rc = lib().q3a_paged_read_fp8(
            k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), k_scale.stride(1), pages, page, slots.data_ptr(),
            k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), T, Hkv, D, _stream(dev))
    check(rc, "q3a_paged_read_fp8")
    return k, v


@paged_read_fp8.register_fake
def _paged_read_fp8_fake(k_cache, v_cache, k_scale, v_scale, slots):
    shape = (slots.shape[0], k_cache.shape[2], k_cache.shape[3])
    return (k_cache.new_empty(shape, dtype=torch.bfloat16), k_cache.new_empty(shape, dtype=torch.bfloat16))


def _check_decode(who, q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table):
    _req(q.is_cuda, f"{who}: tensors must be on a GPU (there is no CPU path)")
    _req(q.dtype == torch.bfloat16 and q.dim() == 3 and q.stride(2) == 1,
         f"{who}: q must be bfloat16 [batch, heads, head_dim] with a contiguous head_dim")
    check_pool(who, q.device, k_cache, v_cache, k_scale, v_scale)
    _req(k_cache.shape[3] == q.shape[2], f"{who}: head_dim mismatch between q and k_cache")
    check_rows(who, q.device, q.shape[0], cache_seqlens, block_table)


def workspace(L, B, N, Hq, Hkv, D, max_pages, page, dev):
    """(workspace or None, its bytes) of a call, from the caching allocator on the current stream."""
    n = L.q3a_paged_decode_tree_workspace_bytes(B, N, Hq, Hkv, D, max_pages, page)
    return (torch.empty((n,), dtype=torch.uint8, device=dev) if n else None), n


@torch.library.custom_op("q3attn::paged_decode_fp8", mutates_args=())
def paged_decode_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                     softmax_scale: float) -> torch.Tensor:
    """``paged_decode`` over the 8-bit pool: o[b, h] = softmax(q[b, h] . K_b^T * scale) . V_b over the cache_seqlens[b] tokens
    of row b, gathered through ``block_table`` [B, max_pages] int32.  q [B, Hq, 128] bf16, Hq a multiple of the pool's KV heads
    (up to 16 times).  Rows with cache_seqlens <= 0 give zeros; table entries outside the pool contribute no tokens."""
    who = "q3attn.paged_decode_fp8"
    _check_decode(who, q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table)
    B, Hq, D = q.shape
    pages, page, Hkv, _ = k_cache.shape
    dev = q.device
    out = torch.empty((B, Hq, D), dtype=q.dtype, device=dev)
    if B == 0:
        return out
    L = lib()
    with torch.cuda.device(dev):
        ws, nbytes = workspace(L, B, 1, Hq, Hkv, D, block_table.shape[1], page, dev)
        rc = L.q3a_paged_decode_fp8(
            q.data_ptr(), q.stride(0), q.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), k_scale.stride(1), pages, page,
            cache_seqlens.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            out.data_ptr(), out.stride(0), out.stride(1), ws.data_ptr() if ws is not None else None, nbytes,
            B, Hq, Hkv, D, float(softmax_scale), _stream(dev))
    check(rc, "q3a_paged_decode_fp8")
    return out


@paged_decode_fp8.register_fake
def _paged_decode_fp8_fake(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale):
    return q.new_empty(q.shape)


@torch.library.custom_op("q3attn::paged_decode_fp8_append", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def paged_decode_fp8_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            k_scale: torch.Tensor, v_scale: torch.Tensor, cache_seqlens: torch.Tensor,
                            block_table: torch.Tensor, softmax_scale: float) -> torch.Tensor:
    """One decode step on the 8-bit pool in one pass: k[b], v[b] [B, Hkv, 128] bf16 (any row and head strides) are quantised
    into position p = cache_seqlens[b] of row b (``paged_write_fp8``'s bytes), and the attention of q[b] over tokens 0..p is
    returned, the new one with the value that the pool now holds (``paged_write_fp8`` then ``paged_decode_fp8``).  Rows with
    cache_seqlens < 0, or without room for the new token, give zeros and write nothing."""
    who = "q3attn.paged_decode_fp8_append"
    _check_decode(who, q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table)
    B, Hq, D = q.shape
    pages, page, Hkv, _ = k_cache.shape
    dev = q.device
    _tokens(who, k, "k", dev)
    _tokens(who, v, "v", dev)
    _req(k.shape == (B, Hkv, D) and v.shape == (B, Hkv, D), f"{who}: k and v must be [{B}, {Hkv}, {D}]")
    out = torch.empty((B, Hq, D), dtype=q.dtype, device=dev)
    if B == 0:
        return out
    L = lib()
    with torch.cuda.device(dev):
        ws, nbytes = workspace(L, B, 1, Hq, Hkv, D, block_table.shape[1], page, dev)
        rc = L.q3a_paged_decode_fp8_append(
            q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
            v.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), k_scale.stride(1), pages, page,
            cache_seqlens.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            out.data_ptr(), out.stride(0), out.stride(1), ws.data_ptr() if ws is not None else None, nbytes,
            B, Hq, Hkv, D, float(softmax_scale), _stream(dev))
    check(rc, "q3a_paged_decode_fp8_append")
    return out


@paged_decode_fp8_append.register_fake
def _paged_decode_fp8_append_fake(q, k, v, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale):
    return q.new_empty(q.shape)
