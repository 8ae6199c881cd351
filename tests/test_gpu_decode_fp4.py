"""Decode attention over the 4-bit pool (plain and append) against attention in 64 bits over the values that the pool holds."""
import math

import numpy as np
import pytest
import torch

import q3attn
from fp4_reference import assert_close, fill_pool, pack, pool_values, quantise, values
from fp8_reference import attention, table_for

pytestmark = pytest.mark.gpu

LENS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 200, 333, 700, -3]


def _case(dev, lens, page, hkv, group, head_major, seed, width=None):
    lens = list(lens)
    used = sum(-(-max(n, 0) // page) for n in lens)
    pool = fill_pool(used + 3, page, hkv, head_major, seed, dev)
    width = max(1, -(-(max(lens) + 1) // page)) if width is None else width
    table = table_for(lens, page, used + 3, width, seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn((len(lens), hkv * group, 128), generator=g).to(torch.bfloat16)
    return pool, table, torch.tensor(lens, dtype=torch.int32), q


def _check(pool, table, lens, q, scale=128 ** -0.5):
    dev = pool[0].device
    out = q3attn.paged_decode_fp4(q.to(dev), *pool, lens.to(dev), table.to(dev), scale)
    want, spread = attention(q[:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, scale)
    assert_close(out, want[:, 0], spread[:, 0])
    return out


@pytest.mark.parametrize("page,hkv,group,head_major", [(16, 8, 2, True), (16, 8, 2, False), (48, 2, 1, True), (64, 4, 4, False),
                                                       (256, 1, 16, True), (16, 3, 3, True),
                                                       (32, 2, 5, False), (16, 4, 8, True)])
def test_ragged_rows(cuda_device, page, hkv, group, head_major):
    _check(*_case(cuda_device, LENS, page, hkv, group, head_major, page + hkv))


@pytest.mark.parametrize("lens", [[2500], [5000, 3], [1, 3000, 40, 0, 1700]])
def test_long_rows_of_small_batches(cuda_device, lens):
    _check(*_case(cuda_device, lens, 16, 8, 2, True, 5))


def test_wide_table(cuda_device):
    """A table much wider than the rows: most of the launch has nothing to do."""
    _check(*_case(cuda_device, [70, 0, 1, 900], 16, 8, 2, True, 6, width=4096))


def test_many_rows(cuda_device):
    rng = np.random.default_rng(7)
    pool, table, lens, q = _case(cuda_device, rng.integers(0, 500, 300), 16, 8, 2, True, 7)
    out = q3attn.paged_decode_fp4(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), 0.09)
    rows = list(range(0, 300, 13))
    want, spread = attention(q[rows][:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens[rows],
                             table[rows], 0.09)
    assert_close(out[rows], want[:, 0], spread[:, 0])


def test_equals_bf16_decode_of_the_values(cuda_device):
    """The values are bf16 numbers, so the bf16 pool's decode over them computes the same attention."""
    pool, table, lens, q = _case(cuda_device, [5, 300, 64, 0, 1000], 16, 8, 2, True, 8)
    slots = torch.arange(pool[0].shape[0] * 16, device=cuda_device)
    k, v = q3attn.paged_read_fp4(*pool, slots)
    args = (lens.to(cuda_device), table.to(cuda_device), 128 ** -0.5)
    a = q3attn.paged_decode_fp4(q.to(cuda_device), *pool, *args)
    b = q3attn.paged_decode(q.to(cuda_device), k.view(-1, 16, 8, 128), v.view(-1, 16, 8, 128), *args)
    _, spread = attention(q[:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, args[2])
    assert_close(a, b.cpu().double(), 2 * spread[:, 0])       # both sides round


def test_what_is_not_attended_does_not_matter(cuda_device):
    """Any codes and exponent bytes (NaN) behind the last token, entries outside the pool, a table behind the row's pages."""
    lens = [5, 37, 16, 70]
    pool, table, lens, q = _case(cuda_device, lens, 16, 8, 2, True, 9, width=7)
    table[1, 1] = 1 << 20                                      # tokens 16..31 of row 1 are gone
    table[3, 0] = -7
    for b, n in enumerate([5, 37, 16, 70]):
        last = int(table[b, (n - 1) // 16])
        if n % 16:
            for t, byte in ((pool[0], 0x7F), (pool[1], 0xFF)):
                t.view(torch.uint8)[last, n % 16:] = byte
            pool[2][last, :, :, n % 16:] = 255
            pool[3][last, :, :, n % 16:] = 255 if b % 2 else 0
    table[0, 1:] = 2
    _check(pool, table, lens, q)


def test_far_scores_and_far_scales(cuda_device):
    """Scores of thousands (one key takes all) and value rows of very different size."""
    pool, table, lens, q = _case(cuda_device, [50, 200], 16, 8, 2, True, 10)
    pool[3].copy_(torch.where(torch.rand(pool[3].shape, generator=torch.Generator().manual_seed(3)).to(cuda_device) < 0.5,
                              pool[3], pool[3] + 40))
    out = q3attn.paged_decode_fp4((q * 64).to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), 1.0)
    want, spread = attention((q * 64)[:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, 1.0)
    # fp32 scores of up to ~2e4: 128 * 2^-24 * 2e4 = 0.15 of a score, so only keys that lead by more than that are certain
    assert torch.isfinite(out.float()).all()
    score_err = 0.17 * 2
    assert_close(out, want[:, 0], spread[:, 0], score_err=score_err)


def test_table_beyond_rows_capacity_is_clamped(cuda_device):
    pool, table, lens, q = _case(cuda_device, [64, 64], 16, 8, 2, True, 11)
    lens = torch.tensor([1000, 70], dtype=torch.int32)         # the table holds 5 pages of which 4 are the row's
    table = table[:, :4].contiguous()
    _check(pool, table, lens, q)


def _append(dev, pool, table, lens, q, k, v, scale=128 ** -0.5):
    return q3attn.paged_decode_fp4_append(q.to(dev), k, v, *pool, lens.to(dev), table.to(dev), scale)


@pytest.mark.parametrize("page,hkv,group,head_major", [(16, 8, 2, True), (64, 4, 4, False), (48, 1, 16, True)])
def test_append_is_write_then_decode(cuda_device, page, hkv, group, head_major):
    """Bytes of the pool exactly those of the write; the result that of 64-bit attention over the pool after it."""
    lens = [0, 1, 15, 16, 31, 32, 47, 48, 100, 700, -1]
    used = [n + 1 for n in lens]
    pool = fill_pool(sum(-(-n // page) for n in used) + 2, page, hkv, head_major, page, cuda_device)
    width = -(-max(used) // page)
    table = table_for(used, page, pool[0].shape[0], width, page)
    g = torch.Generator().manual_seed(page)
    q = torch.randn((len(lens), hkv * group, 128), generator=g).to(torch.bfloat16)
    kv = (torch.randn((len(lens), 2 * hkv, 128), generator=g) * 2).to(torch.bfloat16).to(cuda_device)
    k, v = kv[:, :hkv], kv[:, hkv:]
    lens_t = torch.tensor(lens, dtype=torch.int32)
    other = [t.clone() for t in pool]
    slots = torch.tensor([-1 if n < 0 else int(table[b, n // page]) * page + n % page for b, n in enumerate(lens)])
    q3attn.paged_write_fp4(k, v, slots.to(cuda_device), *other)
    out = _append(cuda_device, pool, table, lens_t, q, k, v)
    torch.cuda.synchronize()
    for a, b in zip(pool, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    want, spread = attention(q[:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]),
                             torch.where(lens_t >= 0, lens_t + 1, lens_t), table, 128 ** -0.5)
    assert_close(out, want[:, 0], spread[:, 0])


def test_append_without_room_or_page(cuda_device):
    pool = fill_pool(8, 16, 8, True, 1, cuda_device)
    before = [t.view(torch.uint8).clone() for t in pool]
    table = torch.tensor([[0, 1], [2, 99], [3, -1], [4, 5]], dtype=torch.int32)
    lens = torch.tensor([32, 20, 16, -5], dtype=torch.int32)   # full; its page invalid (twice); a padded row
    g = torch.Generator().manual_seed(2)
    q = torch.randn((4, 16, 128), generator=g).to(torch.bfloat16)
    k = torch.randn((4, 8, 128), generator=g).to(torch.bfloat16).to(cuda_device)
    out = _append(cuda_device, pool, table, lens, q, k, k)
    torch.cuda.synchronize()
    for a, b in zip(pool, before):
        assert torch.equal(a.view(torch.uint8), b)
    want, spread = attention(q[:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]),
                             torch.tensor([-1, 20, 16, -1]), table, 128 ** -0.5)
    assert_close(out, want[:, 0], spread[:, 0])


def test_append_special_rows(cuda_device):
    """A new row of zeros, of the largest bf16, with NaN: the pool gets the write's bytes, NaN reaches its own row alone."""
    pool = fill_pool(8, 16, 2, True, 4, cuda_device)
    other = [t.clone() for t in pool]
    table = torch.tensor([[0], [1], [2], [3]], dtype=torch.int32)
    lens = torch.tensor([3, 3, 3, 0], dtype=torch.int32)
    k = torch.zeros((4, 2, 128), dtype=torch.bfloat16)
    v = torch.randn((4, 2, 128), generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    v[1, 0, 7] = float("nan")
    v[2, 1] = 3.38953139e38
    v[3] = 0
    q = torch.randn((4, 4, 128), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    out = _append(cuda_device, pool, table, lens, q, k.to(cuda_device), v.to(cuda_device))
    q3attn.paged_write_fp4(k.to(cuda_device), v.to(cuda_device), torch.tensor([3, 19, 35, 48], device=cuda_device), *other)
    for a, b in zip(pool, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    want, spread = attention(q[:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens + 1, table, 128 ** -0.5)
    assert_close(out, want[:, 0], spread[:, 0])
    assert torch.isnan(out[1, 0, 7]) and int(torch.isnan(out).sum()) == 64   # a block of the two query heads of KV head 0


@pytest.mark.parametrize("scale", [0.0, -0.11, 3.0])
def test_any_scale(cuda_device, scale):
    pool, table, lens, q = _case(cuda_device, [1, 40, 333, 0], 16, 2, 4, True, 21)
    _check(pool, table, lens, q, scale)


def test_blocks_and_queries_that_are_not_finite(cuda_device):
    """A NaN block of a key makes its row's heads NaN, one of a value its 32 dims, a query that is not finite its own head."""
    pool, table, lens, q = _case(cuda_device, [20, 50, 64, 33], 16, 2, 2, True, 22)
    pool[2][int(table[0, 1]), 1, 2, 3] = 255                   # key 19 of row 0, KV head 1
    pool[3][int(table[1, 2]), 0, 1, 0] = 255                   # value 32 of row 1, KV head 0, dims 32..63
    q[2, 3, 5] = float("inf")
    q[3, 0, 100] = float("nan")
    out = q3attn.paged_decode_fp4(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), 0.1).cpu()
    nan = torch.zeros(out.shape, dtype=torch.bool)
    nan[0, 2:] = nan[2, 3] = nan[3, 0] = True
    nan[1, :2, 32:64] = True
    assert torch.equal(torch.isnan(out), nan)
    want, spread = attention(q[:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, 0.1)
    want[2, 0, 3] = math.nan                                   # inf - inf in the restatement's softmax, or not, as the signs fall
    assert_close(out, want[:, 0], spread[:, 0])


@pytest.mark.parametrize("rows,hkv,group,most,width", [(65, 1, 2, 300, 4096), (300, 2, 1, 1500, 94), (64, 8, 2, 900, 57), (9, 2, 16, 4000, 260)])
def test_each_form_of_launch(cuda_device, rows, hkv, group, most, width):
    """Chunks of long rows, and whole rows that start in the order of their lengths, with empty ones among them."""
    rng = np.random.default_rng(rows)
    lens = rng.integers(0, most, rows)
    lens[::7] = rng.integers(-2, 3, len(lens[::7]))
    pool, table, lens, q = _case(cuda_device, lens, 16, hkv, group, True, rows, width=width)
    out = q3attn.paged_decode_fp4(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), 0.09)
    pick = sorted({0, 1, 7, rows - 1, *range(2, rows, max(1, rows // 24))})
    want, spread = attention(q[pick][:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens[pick], table[pick], 0.09)
    assert_close(out[pick], want[:, 0], spread[:, 0])
    assert not out[lens <= 0].any()


def test_small_query_elements_count(cuda_device):
    """Keys that are zero where a query's largest element is: its small elements alone make the scores."""
    dev, n = cuda_device, 200
    g = torch.Generator().manual_seed(3)
    k = torch.randn((n, 1, 128), generator=g).to(torch.bfloat16)
    k[..., 5] = 0
    v = torch.randn((n, 1, 128), generator=g).to(torch.bfloat16)
    pool = q3attn.fp4_cache(-(-n // 16), 16, 1, device=dev)
    q3attn.paged_write_fp4(k.to(dev), v.to(dev), torch.arange(n, device=dev), *pool)
    q = torch.randn((1, 2, 128), generator=g).to(torch.bfloat16)
    q[0, 0, 5], q[0, 1, 5] = 2.0 ** 40, -(2.0 ** 100)
    table, lens = torch.arange(-(-n // 16), dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
    _check(pool, table, lens, q)


def test_far_pages(cuda_device):
    """Pages past 4 GiB of codes, and past 2^31 slots of exponent bytes' offsets."""
    dev, pages = cuda_device, 1_200_000
    pool = [torch.empty((pages, 8, 16, 64), dtype=torch.uint8, device=dev).transpose(1, 2) for _ in range(2)]
    pool += [torch.empty((pages, 8, 4, 16), dtype=torch.uint8, device=dev) for _ in range(2)]
    assert pool[0].numel() > 1 << 33
    table = torch.tensor([[pages - 1, 5, pages // 2, pages - 2], [7, pages - 9, -1, -1]], dtype=torch.int32)
    lens = torch.tensor([60, 20], dtype=torch.int32)
    slots = torch.cat([torch.arange(60), 64 + torch.arange(20)])
    slots = table.flatten().long()[slots // 16] * 16 + slots % 16
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn((80, 8, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((2, 16, 128), generator=g).to(torch.bfloat16)
    q3attn.paged_write_fp4(k.to(dev), v.to(dev), slots.to(dev), *pool)
    out = q3attn.paged_decode_fp4(q.to(dev), *pool, lens.to(dev), table.to(dev), 0.1)
    kr, vr = q3attn.paged_read_fp4(*pool, slots.to(dev))
    small = torch.arange(8, dtype=torch.int32).view(2, 4)
    near = [torch.zeros((8 * 16, 8, 128), dtype=torch.float64) for _ in range(2)]
    at = torch.cat([torch.arange(60), 64 + torch.arange(20)])
    near[0][at], near[1][at] = kr.cpu().double(), vr.cpu().double()
    want, spread = attention(q[:, None], near[0].view(8, 16, 8, 128), near[1].view(8, 16, 8, 128), lens, small, 0.1)
    assert_close(out, want[:, 0], spread[:, 0])
    for x, got in ((k, kr), (v, vr)):
        code, byte = quantise(x)
        assert torch.equal(got.cpu().double(), values(pack(code), byte))


@pytest.mark.parametrize("lens", [[900], list(range(0, 640, 8))])
def test_captured_and_replayed(cuda_device, lens):
    pool, table, lens_t, q = _case(cuda_device, lens, 16, 8, 2, True, 12)
    args = (q.to(cuda_device), *pool, lens_t.to(cuda_device), table.to(cuda_device), 128 ** -0.5)
    eager = q3attn.paged_decode_fp4(*args).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q3attn.paged_decode_fp4(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = q3attn.paged_decode_fp4(*args)
    with torch.cuda.graph(second):
        out2 = q3attn.paged_decode_fp4(*args)
    for _ in range(3):
        junk = torch.randn(1 << 18, device=cuda_device) * 3
        out.zero_()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(out2, eager)
        del junk


def test_two_streams(cuda_device):
    cases = [_case(cuda_device, lens, 16, 8, 2, True, 13) for lens in ([2000], [40, 1500, 7])]
    calls = [(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), 0.1) for pool, table, lens, q in cases]
    eager = [q3attn.paged_decode_fp4(*c) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for s, c, g in zip(streams, calls, got):
            with torch.cuda.stream(s):
                g.append(q3attn.paged_decode_fp4(*c))
    torch.cuda.synchronize()
    for g, e in zip(got, eager):
        assert all(torch.equal(x, e) for x in g)


def test_empty_batch(cuda_device):
    pool = q3attn.fp4_cache(2, device=cuda_device)
    out = q3attn.paged_decode_fp4(torch.empty((0, 16, 128), dtype=torch.bfloat16, device=cuda_device), *pool,
                                  torch.empty((0,), dtype=torch.int32, device=cuda_device),
                                  torch.empty((0, 4), dtype=torch.int32, device=cuda_device), 1.0)
    assert out.shape == (0, 16, 128)


def test_refusals(cuda_device):
    pool, table, lens, q = _case(cuda_device, [5, 9], 16, 8, 2, True, 1)
    q, lens, table = q.to(cuda_device), lens.to(cuda_device), table.to(cuda_device)
    bad = [(q.half(), *pool, lens, table), (q[:, :12], *pool, lens, table), (q, *pool, lens.long(), table),
           (q, *pool, lens[:1], table), (q, *pool, lens, table.long()), (q, *pool, lens, table[:1]), (q, *pool, lens.cpu(), table),
           (q, pool[0].view(torch.int8), *pool[1:], lens, table),
           (q, pool[0][..., :32], pool[1][..., :32], *pool[2:], lens, table),
           (q, *pool[:2], pool[2][:, :, :2], pool[3][:, :, :2], lens, table),
           (q, *pool[:2], pool[2].transpose(2, 3).contiguous().transpose(2, 3), pool[3].transpose(2, 3).contiguous().transpose(2, 3), lens,
            table), (q, *pool[:2], pool[2].float(), pool[3].float(), lens, table),
           (torch.zeros((2, 8 * 17, 128), dtype=torch.bfloat16, device=cuda_device), *pool, lens, table),
           (torch.zeros((2, 16, 136), dtype=torch.bfloat16, device=cuda_device)[..., 1:129], *pool, lens, table)]
    for args in bad:
        with pytest.raises(RuntimeError, match="q3a|q3attn"):
            q3attn.paged_decode_fp4(*args, 0.1)
    k = torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=cuda_device)
    for kk, vv in ((k[:1], k), (k, k.float()), (k, k[:, :4])):
        with pytest.raises(RuntimeError, match="q3a|q3attn"):
            q3attn.paged_decode_fp4_append(q, kk, vv, *pool, lens, table, 0.1)


def test_compiled_step_writes_the_callers_pool(cuda_device):
    """Inside torch.compile: the write, the read and the append form mutate the caller's pool in place, without a copy of it."""
    lens = [3, 40, 17]
    pool = q3attn.fp4_cache(4096, device=cuda_device)
    eager_pool = [t.clone() for t in pool]
    table = torch.arange(3 * 4, dtype=torch.int32, device=cuda_device).view(3, 4)
    g = torch.Generator().manual_seed(3)
    q = torch.randn((3, 16, 128), generator=g).to(torch.bfloat16).to(cuda_device)
    k = torch.randn((60, 8, 128), generator=g).to(torch.bfloat16).to(cuda_device)
    slots = torch.cat([torch.arange(n) + 64 * b for b, n in enumerate(lens)]).to(cuda_device)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=cuda_device)

    def step(q, k, kc, vc, ks, vs):
        q3attn.paged_write_fp4(k, k * 2, slots, kc, vc, ks, vs)
        out = q3attn.paged_decode_fp4_append(q + 1, k[:3] - 1, k[3:6], kc, vc, ks, vs, lens_t, table, 0.1)
        return out * 2, q3attn.paged_read_fp4(kc, vc, ks, vs, slots[:5])[0]

    want = step(q, k, *eager_pool)
    compiled = torch.compile(step, dynamic=False)
    compiled(q, k, *[t.clone() for t in pool])
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = compiled(q, k, *pool)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < pool[0].numel() // 2
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, b in zip(pool, eager_pool):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
