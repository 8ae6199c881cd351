"""The 4-bit pool at its limits: offsets of codes and exponent bytes past 2^31 in the units that the kernels count in, pools of 2^31 slots
and more, pools without a page, whole rows of 5 to 8 query heads a KV head in four waves and such as outlast a window of pages, and graphs
whose outputs are cleared before every replay."""
import numpy as np
import pytest
import torch

import q3attn
from fp4_reference import assert_close, pack, pool_values, quantise, values
from fp8_reference import attention
from test_fp4_moves_capi import _decode, _err
from test_gpu_decode_fp4 import _append, _case
from test_gpu_decode_fp4_forms import _far_rows

pytestmark = pytest.mark.gpu


def _write_read_decode(pool, table, lens, group, seed):
    """Rows written at the table's places read back as quantised, and decode (plain, then with a new row) is attention over them."""
    dev, page, hkv = pool[0].device, pool[0].shape[1], pool[0].shape[2]
    rows = [(b, t) for b in range(len(lens)) for t in range(int(lens[b]) + 1)]       # the last one comes with the append form
    slots = torch.tensor([int(table[b, t // page]) * page + t % page for b, t in rows])
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((len(rows), hkv, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((len(lens), hkv * group, 128), generator=g).to(torch.bfloat16)
    last = torch.tensor([i for i, (b, t) in enumerate(rows) if t == int(lens[b])])
    early = torch.ones(len(rows), dtype=torch.bool)
    early[last] = False
    q3attn.paged_write_fp4(k[early].to(dev), v[early].to(dev), slots[early].to(dev), *pool)
    outs = [q3attn.paged_decode_fp4(q.to(dev), *pool, lens.to(dev), table.to(dev), 0.1),
            _append(dev, pool, table, lens, q, k[last].to(dev), v[last].to(dev), 0.1)]
    got = q3attn.paged_read_fp4(*pool, slots.to(dev))
    want = []
    for x, r in zip((k, v), got):
        code, byte = quantise(x)
        want.append(values(pack(code), byte))
        assert torch.equal(r.cpu().double(), want[-1])
    width = table.shape[1]
    small = torch.arange(len(lens) * width, dtype=torch.int32).view(len(lens), width)
    near = [torch.zeros((len(lens) * width * page, hkv, 128), dtype=torch.float64) for _ in range(2)]
    at = torch.tensor([b * width * page + t for b, t in rows])
    for n, w in zip(near, want):
        n[at] = w
    for extra, out in enumerate(outs):
        ref, spread = attention(q[:, None], *(n.view(-1, page, hkv, 128) for n in near), lens + extra, small, 0.1)
        assert_close(out, ref[:, 0], spread[:, 0])
    return slots


@pytest.mark.parametrize("group", [2, 6, 12])                  # each kernel that decodes
def test_exponent_bytes_past_2_to_the_31(cuda_device, group):
    """Scales as a view with pages 512 MiB apart: offsets of up to 3 GiB, of the 4 that are allowed."""
    pages, page, hkv, apart = 7, 16, 2, 1 << 29
    caches = [torch.zeros((pages, page, hkv, 64), dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    scales = [torch.zeros((pages - 1) * apart + hkv * 4 * page, dtype=torch.uint8, device=cuda_device)
              .as_strided((pages, hkv, 4, page), (apart, 4 * page, page, 1)) for _ in range(2)]
    table = torch.tensor([[6, 0, 4], [1, 5, -1]], dtype=torch.int32)
    assert int(table.max()) * apart > 1 << 31
    _write_read_decode([*caches, *scales], table, torch.tensor([40, 20], dtype=torch.int32), group, group)


@pytest.mark.parametrize("group", [1, 8, 16])
def test_codes_past_2_to_the_31_units(cuda_device, group):
    """Caches as views with pages 8 GiB apart, K's and V's in the same memory: offsets of 32 GiB and more, 2^31 times 16 bytes."""
    pages, page, hkv, apart = 5, 32, 1, 1 << 33
    memory = torch.empty((pages - 1) * apart + (2 << 20), dtype=torch.uint8, device=cuda_device)
    caches = [memory.as_strided((pages, page, hkv, 64), (apart, 64, 64, 1), i << 20) for i in range(2)]
    scales = [torch.zeros((pages, hkv, 4, page), dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    table = torch.tensor([[4, 0, 2], [1, 3, -1]], dtype=torch.int32)
    assert int(table.max()) * apart >= 16 << 31
    _write_read_decode([*caches, *scales], table, torch.tensor([70, 35], dtype=torch.int32), group, group)


@pytest.mark.parametrize("page", [16, 48])
def test_pool_of_2_to_the_31_slots(cuda_device, page):
    """Pages 16 bytes of codes and 4 of exponents apart, of which few are used, far from each other: slots past 2^31."""
    pages, hkv = (1 << 31) // page + 900, 1
    caches = [torch.zeros(16 * pages + 64 * page, dtype=torch.uint8, device=cuda_device)
              .as_strided((pages, page, hkv, 64), (16, 64, 64, 1)) for _ in range(2)]
    scales = [torch.zeros(4 * pages + 4 * page, dtype=torch.uint8, device=cuda_device)
              .as_strided((pages, hkv, 4, page), (4, 4 * page, page, 1)) for _ in range(2)]
    far = pages - 1
    table = torch.tensor([[far, 0, far - 400], [pages // 2, far - 800, 400]], dtype=torch.int32)
    slots = _write_read_decode([*caches, *scales], table, torch.tensor([2 * page + 5, page + 9], dtype=torch.int32), 2, page)
    assert int(slots.max()) >= 1 << 31
    assert int(slots.max()) // page == far


@pytest.mark.parametrize("rows,hkv,group,head_major", [(80, 4, 8, True), (80, 4, 5, False), (300, 1, 7, True), (50, 8, 6, False)])
@pytest.mark.parametrize("append", [False, True])
def test_whole_rows_of_5_to_8_heads_in_four_waves(cuda_device, rows, hkv, group, head_major, append):
    """More (row, KV head) pairs than compute units, with rows of no token and of all that the table holds among them."""
    rng = np.random.default_rng(rows + group)
    lens = rng.integers(0, 200, rows)
    lens[::9] = rng.integers(700, 959, len(lens[::9]))
    lens[4::11] = rng.integers(-2, 2, len(lens[4::11]))
    pool, table, _, q = _case(cuda_device, [n + 1 for n in lens], 16, hkv, group, head_major, rows + group, width=60)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    g = torch.Generator().manual_seed(rows)
    if append:
        k, v = (torch.randn((rows, hkv, 128), generator=g).to(torch.bfloat16).to(cuda_device) for _ in range(2))
        out = _append(cuda_device, pool, table, lens_t, q, k, v)
        lens_t = torch.where(lens_t >= 0, lens_t + 1, -1)
    else:
        out = q3attn.paged_decode_fp4(q.to(cuda_device), *pool, lens_t.to(cuda_device), table.to(cuda_device), 128 ** -0.5)
    pick = sorted({0, rows - 1, *range(0, rows, max(9, 9 * (rows // 150))), *range(4, min(rows, 40), 11), *range(1, rows, 13)})
    want, spread = attention(q[pick][:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens_t[pick], table[pick], 128 ** -0.5)
    assert_close(out[pick], want[:, 0], spread[:, 0])
    assert not out[lens_t <= 0].any() and torch.isfinite(out.float()).all()


@pytest.mark.parametrize("group", [2, 6])
@pytest.mark.parametrize("append", [False, True])
def test_whole_rows_that_outlast_a_window(cuda_device, group, append):
    """A row of more than 4096 tokens, where four waves look up their pages again, in a batch that is not cut into chunks."""
    rng = np.random.default_rng(group)
    _far_rows(cuda_device, [4500] + [int(n) for n in rng.integers(1, 60, 199)], 8, group, 290, 40 + group, append)


@pytest.mark.parametrize("rows,hq,hkv,max_pages", [(3, 16, 8, 6), (3, 56, 8, 6), (3, 128, 8, 6), (70, 8, 4, 6), (70, 28, 4, 6),
                                                   (3, 16, 8, 4096), (3, 56, 8, 4096), (3, 128, 8, 4096)])
@pytest.mark.parametrize("append", [False, True])
def test_pool_without_pages_at_the_c_entry(cuda_device, rows, hq, hkv, max_pages, append):
    """No page, but memory to point to: every row is zeros, whatever the lengths and the table say, and nothing is written."""
    dev = cuda_device
    memory = [torch.full((4096,), 119, dtype=torch.uint8, device=dev) for _ in range(4)]
    f = lambda heads: torch.ones((rows, heads, 128), dtype=torch.bfloat16, device=dev)
    q, k, v, out = f(hq), f(hkv), f(hkv), f(hq)
    lens = torch.tensor([5, 0, 70, 3] * 20, dtype=torch.int32, device=dev)[:rows].contiguous()
    table = torch.full((rows, max_pages), 2, dtype=torch.int32, device=dev)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    rc = _decode(append, pages=0, kc=memory[0].data_ptr(), vc=memory[1].data_ptr(), ks=memory[2].data_ptr(), vs=memory[3].data_ptr(),
                 q=q.data_ptr(), q_sb=q.stride(0), kn=k.data_ptr(), kn_sb=k.stride(0), vn=v.data_ptr(), vn_sb=v.stride(0), lens=lens.data_ptr(),
                 bt=table.data_ptr(), bt_sb=max_pages, max_pages=max_pages, out=out.data_ptr(), o_sb=out.stride(0), ws=ws.data_ptr(),
                 ws_bytes=ws.numel(), B=rows, Hq=hq, Hkv=hkv)
    assert rc == 0, _err()
    torch.cuda.synchronize()
    assert not out.any()
    assert all(bool((m == 119).all()) for m in memory)


@pytest.mark.parametrize("lens", [[900], list(range(0, 640, 8)), [3000, 40]])
@pytest.mark.parametrize("group", [2, 7])
def test_graphs_that_share_their_memory_write_again(cuda_device, lens, group):
    """Two graphs of one memory, both outputs cleared before every replay."""
    pool, table, lens_t, q = _case(cuda_device, lens, 16, 8, group, True, 12 + group)
    args = (q.to(cuda_device), *pool, lens_t.to(cuda_device), table.to(cuda_device), 128 ** -0.5)
    eager = q3attn.paged_decode_fp4(*args).clone()
    graphs, outs, shared = [], [], None
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=shared):
            outs.append(q3attn.paged_decode_fp4(*args))
        shared = graph.pool()
        graphs.append(graph)
    for _ in range(3):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, out in zip(graphs, outs):
            graph.replay()
            junk = torch.randn(1 << 18, device=cuda_device) * 3      # the program's own work between replays
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
            del junk
        assert torch.equal(outs[0], eager)
