"""Decode over the 4-bit pool: rows so long that a wave looks up its pages again, queries of every range, and every ratio of heads, in
every form of launch."""
import math

import numpy as np
import pytest
import torch

import q3attn
from fp4_reference import assert_close, fill_pool, pool_values, values
from fp8_reference import attention, table_for
from test_gpu_decode_fp4 import LENS, _append, _case, _check

pytestmark = pytest.mark.gpu


def _far_rows(dev, lens, hkv, group, width, seed, append):
    """Random codes and exponents on the device; the 64-bit result for some rows and heads alone."""
    g = torch.Generator(device=dev).manual_seed(seed)
    page, used = 16, [-(-max(n + 1, 0) // 16) for n in lens]
    pages = sum(used) + 2
    pool = [torch.randint(0, 256, (pages, hkv, page, 64), generator=g, device=dev, dtype=torch.uint8).transpose(1, 2) for _ in range(2)]
    pool += [torch.randint(120, 126, (pages, hkv, 4, page), generator=g, device=dev, dtype=torch.uint8) for _ in range(2)]
    table = table_for([n + 1 for n in lens], page, pages, width, seed)
    q = torch.randn((len(lens), hkv * group, 128), generator=g, device=dev).to(torch.bfloat16)
    args = (torch.tensor(lens, dtype=torch.int32, device=dev), table.to(dev), 0.05)
    if append:
        k, v = (torch.randn((len(lens), hkv, 128), generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
        out = q3attn.paged_decode_fp4_append(q, k, v, *pool, *args)
    else:
        out = q3attn.paged_decode_fp4(q, *pool, *args)
    torch.cuda.synchronize()
    n = torch.tensor(lens) + int(append)
    rows = sorted(range(len(lens)), key=lambda b: -lens[b])[:2] + [len(lens) - 1]
    for b in rows:
        for h in {0, hkv - 1}:
            ids = table[b, :-(-int(n[b]) // page)].long().to(dev)
            kv = [values(pool[i][ids, :, h].cpu(), pool[2 + i][ids, h].transpose(1, 2).cpu()).reshape(-1, 128)[:int(n[b])] for i in range(2)]
            heads = slice(h * group, (h + 1) * group)
            p = torch.softmax(q[b, heads].cpu().double() @ kv[0].T * 0.05, -1)
            # sums of more terms than assert_close's 5000: 2^-24 each
            assert_close(out[b, heads], p @ kv[1], p @ kv[1].abs(), score_err=5e-4 + n[b].item() * 2.0 ** -24)


# whole rows; chunks of four waves; chunks of eight
@pytest.mark.parametrize("rows,hkv,group,longest,width", [(200, 8, 2, 4500, 400), (1, 64, 1, 68000, 4300), (1, 64, 6, 68000, 4300)])
@pytest.mark.parametrize("append", [False, True])
def test_rows_that_outlast_a_window(cuda_device, rows, hkv, group, longest, width, append):
    rng = np.random.default_rng(rows)
    lens = [longest] + [int(n) for n in rng.integers(1, 60, rows - 1)]
    _far_rows(cuda_device, lens, hkv, group, width, rows + group, append)


@pytest.mark.parametrize("group", [6, 7])
def test_other_ratios_of_heads_and_strided_pools(cuda_device, group):
    """Pools that are some heads of a larger one, token-major."""
    pool, table, lens, q = _case(cuda_device, LENS, 32, 3, group, False, group)
    wide = [torch.zeros((t.shape[0], 32, 5, 64), dtype=torch.uint8, device=cuda_device) for t in pool[:2]]
    for w, t in zip(wide, pool):
        w[:, :, 1:4] = t
    _check((wide[0][:, :, 1:4], wide[1][:, :, 1:4], *pool[2:]), table, lens, q)


@pytest.mark.parametrize("group,lens", [(2, [300, 40]), (7, [70, 129]), (2, [7000]), (5, [5000])])
@pytest.mark.parametrize("append", [False, True])
def test_queries_of_a_wide_range(cuda_device, group, lens, append):
    """Elements 2^30 and more below their block's largest one, that keys of 0 there leave as all that counts; and not finite ones."""
    dev, hkv = cuda_device, 2
    pool = fill_pool(sum(-(-(n + 1) // 16) for n in lens) + 2, 16, hkv, True, 3, dev)
    pool[0][..., 10] = 0                                      # dims 20 and 21 of every key
    table = table_for([n + 1 for n in lens], 16, pool[0].shape[0], max(-(-(n + 1) // 16) for n in lens), 4)
    g = torch.Generator().manual_seed(group)
    q = torch.randn((len(lens), hkv * group, 128), generator=g).to(torch.bfloat16)
    q[..., 20] = torch.randn(q.shape[:2], generator=g).to(torch.bfloat16) * 2.0 ** 45
    q[0, 0, 40] = 2.0 ** -60
    lens_t = torch.tensor(lens, dtype=torch.int32)
    if not append:
        _check(pool, table, lens_t, q)
        return
    kv = torch.randn((len(lens), 2 * hkv, 128), generator=g).to(torch.bfloat16)
    kv[..., 20:22] = 0
    kv = kv.to(dev)
    out = _append(dev, pool, table, lens_t, q, kv[:, :hkv], kv[:, hkv:])
    want, spread = attention(q[:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens_t + 1, table, 128 ** -0.5)
    assert_close(out, want[:, 0], spread[:, 0])
    q[0, 1, 77] = math.inf
    out = _append(dev, pool, table, lens_t, q, kv[:, :hkv], kv[:, hkv:]).cpu()
    assert torch.isnan(out[0, 1]).all() and int(torch.isnan(out).sum()) == 128


def test_every_place_of_the_new_row(cuda_device):
    """Its token first, last or anywhere in a subtile, a step and a page: 130 rows of 0 to 129 tokens before it."""
    dev, lens = cuda_device, list(range(130))
    pool = fill_pool(sum(-(-(n + 1) // 32) for n in lens) + 2, 32, 2, True, 5, dev)
    table = table_for([n + 1 for n in lens], 32, pool[0].shape[0], 5, 6)
    g = torch.Generator().manual_seed(7)
    q = torch.randn((130, 4, 128), generator=g).to(torch.bfloat16)
    k, v = (torch.randn((130, 2, 128), generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    lens_t = torch.tensor(lens, dtype=torch.int32)
    other = [t.clone() for t in pool]
    slots = torch.tensor([int(table[b, b // 32]) * 32 + b % 32 for b in lens], device=dev)
    q3attn.paged_write_fp4(k, v, slots, *other)
    out = _append(dev, pool, table, lens_t, q, k, v)
    for a, b in zip(pool, other):
        assert torch.equal(a, b)
    want, spread = attention(q[:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens_t + 1, table, 128 ** -0.5)
    assert_close(out, want[:, 0], spread[:, 0])


def test_pool_without_pages(cuda_device):
    dev = cuda_device
    pool = q3attn.fp4_cache(0, device=dev)
    q = torch.ones((3, 16, 128), dtype=torch.bfloat16, device=dev)
    lens, table = torch.tensor([5, 0, 70], dtype=torch.int32, device=dev), torch.full((3, 6), 2, dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="null pool"):
        q3attn.paged_decode_fp4(q, *pool, lens, table, 0.1)


@pytest.mark.parametrize("group", [2, 7])
def test_chunks_captured_on_two_streams(cuda_device, group):
    """Chunks and their join in two graphs that share their memory, replayed in turn and with eager calls on another stream between."""
    cases = [_case(cuda_device, lens, 16, 8, group, True, 31 + group) for lens in ([2600], [40, 3100, 7])]
    calls = [(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), 0.1) for pool, table, lens, q in cases]
    eager = [q3attn.paged_decode_fp4(*c).clone() for c in calls]
    graphs, outs, pool = [], [], None
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(q3attn.paged_decode_fp4(*c))
        pool = graph.pool()
        graphs.append(graph)
    side = torch.cuda.Stream()
    for _ in range(4):
        for graph, out, want, call in zip(graphs, outs, eager, calls):
            graph.replay()
            with torch.cuda.stream(side):
                beside = q3attn.paged_decode_fp4(*call)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(beside, want)
