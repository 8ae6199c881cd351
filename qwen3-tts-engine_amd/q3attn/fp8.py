"""The 8-bit K/V pool as torch ops over the q3attn C ABI: its buffers, the quantising write, the read back, and decode
attention over it.

A pool row (one token of one KV head, 128 values) is held as e4m3 codes and one exponent byte s, value = code * 2^(s - 127):
the smallest power of two that takes the row's largest finite magnitude to at most 448 (at least 2^-117; elements that are not
finite are held as NaN).  A row takes 129 bytes instead of 256.  The scale being a power of two, every value read back is a bf16
number, and attention over the pool is attention over the bf16 rows that ``paged_read_fp8`` returns.

The ops are registered from C++ (binding/torch_ops.cpp), where their arguments are checked, enqueue on the tensors' device's
current stream, allocate only through torch's caching allocator and never synchronise.  GPU only.  None has a backward (one that is
asked for raises), and those that write into caches count as in-place operations on them.
"""
from __future__ import annotations

import torch

from ._lib import torch_op

E4M3 = torch.float8_e4m3fn


def _read_fake(k_cache, v_cache, k_scale, v_scale, slots):
    shape = (slots.shape[0], k_cache.shape[2], k_cache.shape[3])
    return (k_cache.new_empty(shape, dtype=torch.bfloat16), k_cache.new_empty(shape, dtype=torch.bfloat16))


_write = torch_op("paged_write_fp8", lambda k, v, slots, k_cache, v_cache, k_scale, v_scale: None)
_read = torch_op("paged_read_fp8", _read_fake)
_decode = torch_op("paged_decode_fp8", lambda q, *rest: q.new_empty(q.shape))
_decode_append = torch_op("paged_decode_fp8_append", lambda q, *rest: q.new_empty(q.shape))


def fp8_cache(num_pages: int, page_size: int = 16, num_kv_heads: int = 8, head_dim: int = 128, device="cuda"):
    """Buffers of one layer's 8-bit pool: (k_cache, v_cache, k_scale, v_scale), k/v_cache [num_pages, page_size, kv_heads,
    head_dim] float8_e4m3fn and k/v_scale [num_pages, kv_heads, page_size] uint8, all holding the value 0.  The caches are
    views whose memory holds a page's tokens of one head next to each other, so a head's page is one run of memory; the ops
    take any strides."""
    caches = [torch.zeros((num_pages, num_kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(E4M3)
              .transpose(1, 2) for _ in range(2)]
    scales = [torch.full((num_pages, num_kv_heads, page_size), 127, dtype=torch.uint8, device=device) for _ in range(2)]
    return (*caches, *scales)


def paged_write_fp8(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Quantise rows k, v [T, Hkv, 128] bf16 (any token and head strides) into the 8-bit pool: token t at ``slots[t]`` = page *
    page_size + offset (int64, as ``PagePool.slot`` gives them); a slot outside the pool (-1) is not written.  A slot given to
    two tokens holds a mix of both afterwards, so only a scratch slot that nothing reads may be given twice.  For this pool
    what the index_copy_ pair of engine/talker.py:72-73 and :161-162 is for the bf16 one."""
    _write(k, v, slots, k_cache, v_cache, k_scale, v_scale)


def paged_read_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                   slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows of ``slots`` [T] int64 as (k, v) [T, Hkv, 128] bf16, exactly as the pool holds them: the packed K/V that
    ``flash_attn_varlen_func`` takes, for a prefill over a cached prefix.  Slots outside the pool (-1) read zeros."""
    return _read(k_cache, v_cache, k_scale, v_scale, slots)


def paged_decode_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                     softmax_scale: float) -> torch.Tensor:
    """``paged_decode`` over the 8-bit pool: o[b, h] = softmax(q[b, h] . K_b^T * scale) . V_b over the cache_seqlens[b] tokens
    of row b, gathered through ``block_table`` [B, max_pages] int32.  q [B, Hq, 128] bf16, Hq a multiple of the pool's KV heads
    (up to 16 times).  Rows with cache_seqlens <= 0 give zeros; table entries outside the pool contribute no tokens."""
    return _decode(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale)


def paged_decode_fp8_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            k_scale: torch.Tensor, v_scale: torch.Tensor, cache_seqlens: torch.Tensor,
                            block_table: torch.Tensor, softmax_scale: float) -> torch.Tensor:
    """One decode step on the 8-bit pool in one pass: k[b], v[b] [B, Hkv, 128] bf16 (any row and head strides) are quantised
    into position p = cache_seqlens[b] of row b (``paged_write_fp8``'s bytes), and the attention of q[b] over tokens 0..p is
    returned, the new one with the value that the pool now holds (``paged_write_fp8`` then ``paged_decode_fp8``).  Rows with
    cache_seqlens < 0, or without room for the new token, give zeros and write nothing."""
    return _decode_append(q, k, v, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale)
