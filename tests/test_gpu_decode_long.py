"""Decode over the 8-bit pool and attention for trees over rows so long that a wave looks up its page ids more than once (a wave
holds those of 32 of its steps, every fourth step of 32 tokens being one wave's: 4096 tokens of a whole row or of a chunk)."""
import pytest
import torch

import q3attn
from fp8_reference import D, assert_close, attention, pool_values
from q3attn import _lib
from test_gpu_decode_tree import _tree_masks

pytestmark = pytest.mark.gpu

SCALE = D ** -0.5


def _pool(dev, lens, page, hkv, fp8, seed, width):
    """Random rows in a pool of fewer pages than the rows have (they share them, in another order each, but for a row's last page),
    and the table."""
    shared = 24 * 1024 // page
    pages = shared + len(lens)
    g = torch.Generator(device=dev).manual_seed(seed)
    kv = [torch.randn((pages * page, hkv, D), generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2)]
    if fp8:
        pool = q3attn.fp8_cache(pages, page, hkv, device=dev)
        q3attn.paged_write_fp8(*kv, torch.arange(pages * page, device=dev), *pool)
    else:
        pool = (kv[0].view(pages, page, hkv, D), kv[1].view(pages, page, hkv, D), None, None)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        used = -(-max(n, 0) // page)
        if used:
            order = [torch.randperm(shared, generator=torch.Generator().manual_seed(seed + 100 * b + i)) for i in range(-(-used // shared))]
            table[b, :used] = torch.cat(order)[:used]
            table[b, used - 1] = shared + b
    return pool, table


def _is_chunked(lens, N, hq, hkv, width, page):
    return _lib.lib().q3a_paged_decode_tree_workspace_bytes(len(lens), N, hq, hkv, D, width, page) > 0


def _check(pool, table, lens, q, out, rows, heads, group, own=None):
    """Rows and KV heads of a result [B, N, Hq, D]; own = (k, v, mask) of the nodes."""
    part = lambda c, s: pool_values(c[:, :, heads], None if s is None else s[:, heads].contiguous())
    qh = [h * group + i for h in heads for i in range(group)]
    more = None if own is None else (own[0][rows][:, :, heads], own[1][rows][:, :, heads], own[2][rows])
    want, spread = attention(q[rows][:, :, qh], part(pool[0], pool[2]), part(pool[1], pool[3]), [lens[b] for b in rows], table[rows],
                             SCALE, more)
    assert_close(out[rows][:, :, qh], want, spread)


def _rows(n, hq, hkv, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((*n, h, D), generator=g).to(torch.bfloat16) for h in (hq, hkv, hkv)]


EDGES = [4096, 4097, 4128, 4129, 8193, 9000]


@pytest.mark.parametrize("page", [16, 48])
def test_whole_rows_of_many_heads(cuda_device, page):
    """48 rows, 64 KV heads: enough workgroups for whole rows in a table of 9024 tokens; plain, appending, and trees of 3 nodes."""
    dev, hkv = cuda_device, 64
    lens = EDGES + [1, 0, -1] + [7 * i for i in range(39)]
    width = 9024 // page
    rows, heads = [0, 1, 2, 3, 4, 5, 6, 20, 47], [0, 37]
    pool, table = _pool(dev, [n + 1 for n in lens], page, hkv, True, 1, width)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    dl, dt = lens_t.to(dev), table.to(dev)
    assert not _is_chunked(lens, 1, hkv, hkv, width, page) and not _is_chunked(lens, 3, hkv, hkv, width, page)
    q, k, v = _rows((48, 3), hkv, hkv, 2)
    mask = _tree_masks(48, 3, 3)
    dq, dk, dv = q.to(dev), k.to(dev), v.to(dev)
    out = q3attn.paged_decode_tree(dq, dk, dv, mask.to(dev), pool[0], pool[1], dl, dt, SCALE, pool[2], pool[3])
    _check(pool, table, lens, q, out, rows, heads, 1, (k, v, mask))
    out = q3attn.paged_decode_fp8(dq[:, 0], *pool, dl, dt, SCALE)
    _check(pool, table, lens, q[:, :1], out[:, None], rows, heads, 1)
    out = q3attn.paged_decode_fp8_append(dq[:, 0], dk[:, 0], dv[:, 0], *pool, dl, dt, SCALE)
    now = [n + 1 if n >= 0 else n for n in lens]
    _check(pool, table, now, q[:, :1], out[:, None], rows, heads, 1)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("n", [4097, 4129, 9000])
def test_whole_rows_of_wide_trees(cuda_device, fp8, n):
    """64 nodes of 256 heads over 16 KV heads: 512 workgroups a row."""
    dev, N, hq, hkv, width = cuda_device, 64, 256, 16, 600
    pool, table = _pool(dev, [n], 16, hkv, fp8, 4, width)
    assert not _is_chunked([n], N, hq, hkv, width, 16)
    q, k, v = _rows((1, N), hq, hkv, 5)
    mask = _tree_masks(1, N, 6)
    out = q3attn.paged_decode_tree(q.to(dev), k.to(dev), v.to(dev), mask.to(dev), pool[0], pool[1],
                                   torch.tensor([n], dtype=torch.int32, device=dev), table.to(dev), SCALE, pool[2], pool[3])
    nodes = [0, 31, 63]
    _check(pool, table, [n], q[:, nodes], out[:, nodes], [0], [0, 15], 16, (k, v, mask[:, nodes]))


@pytest.mark.parametrize("fp8", [True, False])
def test_whole_rows_of_small_trees(cuda_device, fp8):
    dev, hkv, page = cuda_device, 64, 16
    lens = EDGES + [5] * 42
    width = 9024 // page
    pool, table = _pool(dev, lens, page, hkv, fp8, 7, width)
    assert not _is_chunked(lens, 2, hkv, hkv, width, page)
    q, k, v = _rows((48, 2), hkv, hkv, 8)
    mask = _tree_masks(48, 2, 9)
    out = q3attn.paged_decode_tree(q.to(dev), k.to(dev), v.to(dev), mask.to(dev), pool[0], pool[1],
                                   torch.tensor(lens, dtype=torch.int32, device=dev), table.to(dev), SCALE, pool[2], pool[3])
    _check(pool, table, lens, q, out, [0, 1, 2, 3, 4, 5, 20], [1, 63], 1, (k, v, mask))


# 64 KV heads leave 8 chunks of a row (4 with two blocks of query rows): of 33 rounds of 128 tokens from 256 rounds on, and of 40
@pytest.mark.parametrize("n", [32768, 32769, 33792, 40001])
def test_chunks_of_decode(cuda_device, n):
    dev, hkv, page = cuda_device, 64, 16
    width = 40960 // page
    pool, table = _pool(dev, [n + 1], page, hkv, True, 10, width)
    assert _is_chunked([n], 1, hkv, hkv, width, page)
    q, k, v = _rows((1, 1), hkv, hkv, 11)
    lens, dt = torch.tensor([n], dtype=torch.int32, device=dev), table.to(dev)
    out = q3attn.paged_decode_fp8(q[:, 0].to(dev), *pool, lens, dt, SCALE)
    _check(pool, table, [n], q, out[:, None], [0], [0, 40], 1)
    out = q3attn.paged_decode_fp8_append(q[:, 0].to(dev), k[:, 0].to(dev), v[:, 0].to(dev), *pool, lens, dt, SCALE)
    _check(pool, table, [n + 1], q, out[:, None], [0], [0, 40], 1)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("n,N", [(32769, 3), (40001, 3), (20000, 40), (16385, 40)])
def test_chunks_of_trees(cuda_device, fp8, n, N):
    dev, hkv, page = cuda_device, 64, 16
    width = 40960 // page
    pool, table = _pool(dev, [n], page, hkv, fp8, 12, width)
    assert _is_chunked([n], N, hkv, hkv, width, page)
    q, k, v = _rows((1, N), hkv, hkv, 13)
    mask = _tree_masks(1, N, 14)
    out = q3attn.paged_decode_tree(q.to(dev), k.to(dev), v.to(dev), mask.to(dev), pool[0], pool[1],
                                   torch.tensor([n], dtype=torch.int32, device=dev), table.to(dev), SCALE, pool[2], pool[3])
    nodes = sorted({0, 1, N - 1})
    _check(pool, table, [n], q[:, nodes], out[:, nodes], [0], [0, 40], 1, (k, v, mask[:, nodes]))
