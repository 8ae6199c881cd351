"""Decode over the 8-bit pool and attention for trees where the launch takes another form: chunks of long rows in batches of any
size, whole rows that start in the order of their lengths, far pages, odd scales and queries, graphs that share their memory."""
import numpy as np
import pytest
import torch

import q3attn
from fp8_reference import D, E4M3, assert_close, attention, fill_pool, pool_values, quantise, table_for
from test_gpu_decode_fp8 import _case as decode_case
from test_gpu_decode_tree import _case as tree_case, _run as run_tree, _tree_masks

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def _check_rows(pool, table, lens, q, out, rows, scale=SCALE):
    want, spread = attention(q[rows][:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens[rows],
                             table[rows], scale)
    assert_close(out[rows], want[:, 0], spread[:, 0])


def _ragged(rows, most, seed):
    lens = np.random.default_rng(seed).integers(0, most, rows)
    lens[:: 7] = np.random.default_rng(seed).integers(-2, 3, len(lens[:: 7]))
    return lens


@pytest.mark.parametrize("rows,hkv,most,width", [(65, 1, 300, 4096), (130, 2, 200, 2048), (1024, 1, 60, 512), (63, 8, 400, 600)])
def test_chunks_of_many_rows(cuda_device, rows, hkv, most, width):
    """Tables much longer than the chip would like a row to be, most rows short, some of them long."""
    lens = _ragged(rows, most, rows)
    lens[[3, rows // 2, rows - 1]] = [5 * most, 1, 8 * most]
    pool, table, lens, q = decode_case(cuda_device, lens, 16, hkv, 2, True, rows, width=width)
    assert 16 * width * 256 > 512 * (256 + rows * hkv)
    out = q3attn.paged_decode_fp8(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), SCALE)
    pick = sorted({0, 3, 7, rows // 2, rows - 1, *range(1, rows, max(1, rows // 40))})
    _check_rows(pool, table, lens, q, out, pick)
    assert not out[lens <= 0].any()


@pytest.mark.parametrize("rows,hkv,most", [(5, 64, 900), (64, 8, 900), (256, 2, 1000), (300, 2, 1500), (520, 1, 1400)])
def test_rows_in_the_order_of_their_lengths(cuda_device, rows, hkv, most):
    lens = _ragged(rows, most, rows)
    pool, table, lens, q = decode_case(cuda_device, lens, 16, hkv, 1, True, rows, width=-(-most // 16))
    assert rows * hkv > 256 and most * 256 <= 512 * (256 + rows * hkv)
    out = q3attn.paged_decode_fp8(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), SCALE)
    pick = sorted({0, 1, rows - 1, *range(2, rows, max(1, rows // 40))})
    _check_rows(pool, table, lens, q, out, pick)
    assert not out[lens <= 0].any()
    # every row is some workgroup's, whatever the order: the same rows alone, as far as a coarse look tells
    lone = torch.cat([q3attn.paged_decode_fp8(q[i:i + 1].to(cuda_device), *pool, lens[i:i + 1].to(cuda_device),
                                              table[i:i + 1].to(cuda_device), SCALE) for i in range(rows)])
    a, b = out.double(), lone.double()
    assert ((a - b).abs() <= 2.0 ** -6 * b.abs() + 0.05).all() and torch.equal(lens.to(cuda_device) <= 0, ~b.flatten(1).any(1))


@pytest.mark.parametrize("rows,hkv,width", [(130, 1, 2048), (300, 2, 80)])
def test_append_to_many_rows(cuda_device, rows, hkv, width):
    lens = _ragged(rows, 300, rows)
    lens[5] = 16 * width                                       # no room: skipped
    grown = [0 if n < 0 or n == 16 * width else int(n) + 1 for n in lens]
    used = sum(-(-n // 16) for n in grown)
    pool = fill_pool(used + 3, 16, hkv, True, True, rows, cuda_device)
    table = table_for(grown, 16, used + 3, width, rows)
    g = torch.Generator().manual_seed(rows)
    q = torch.randn((rows, 2 * hkv, D), generator=g).to(torch.bfloat16)
    k, v = (torch.randn((rows, hkv, D), generator=g).to(torch.bfloat16) for _ in range(2))
    lens = torch.from_numpy(lens).to(torch.int32)
    out = q3attn.paged_decode_fp8_append(q.to(cuda_device), k.to(cuda_device), v.to(cuda_device), *pool, lens.to(cuda_device),
                                         table.to(cuda_device), SCALE)
    now = torch.tensor(grown, dtype=torch.int32)
    live = [i for i in range(rows) if grown[i] > 0]
    for x, cache, scale in ((k, pool[0], pool[2]), (v, pool[1], pool[3])):
        code, byte = quantise(x)
        vals = pool_values(cache, scale)
        for i in live:
            got = vals[int(table[i, (grown[i] - 1) // 16]), (grown[i] - 1) % 16]
            assert torch.equal(got, code[i] * torch.exp2(byte[i].double() - 127)[:, None])
    pick = live[:: max(1, rows // 40)] + [5]
    _check_rows(pool, table, now, q, out, pick)
    assert not out[now <= 0].any()


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("lens,N,hkv,group", [([2000, 5, 700], 40, 2, 2), ([3000], 130, 1, 1), ([0, 1500, -1, 33], 17, 3, 2),
                                              ([900, 0, 2500], 3, 1, 16)])
def test_chunks_of_trees(cuda_device, fp8, lens, N, hkv, group):
    """Several blocks of query rows over rows of several chunks, whose last one has the own keys."""
    case = tree_case(cuda_device, lens, N, 16, hkv, group, fp8, True, N)
    mask = _tree_masks(len(lens), N, N)
    out = run_tree(cuda_device, *case, mask)
    pool, table, lens, q, k, v = case
    nodes = sorted({0, 1, N // 2, N - 1, *range(0, N, 11)})
    want, spread = attention(q[:, nodes], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, SCALE,
                             (k, v, mask[:, nodes]))
    assert_close(out[:, nodes], want, spread)


@pytest.mark.parametrize("fp8", [True, False])
def test_trees_of_many_rows(cuda_device, fp8):
    lens = _ragged(270, 700, 1).tolist()
    pool, table, lens, q, k, v = tree_case(cuda_device, lens, 3, 16, 2, 2, fp8, True, 4, width=48)
    mask = _tree_masks(270, 3, 5)
    out = run_tree(cuda_device, pool, table, lens, q, k, v, mask)
    pick = list(range(0, 270, 9)) + [269]
    want, spread = attention(q[pick], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens[pick], table[pick], SCALE,
                             (k[pick], v[pick], mask[pick]))
    assert_close(out[pick], want, spread)
    assert not out[lens < 0].any()


@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("lens", [[200, 1, 33], [1500]])
def test_scales_that_are_not_positive(cuda_device, scale, lens):
    pool, table, lens_t, q = decode_case(cuda_device, lens, 16, 2, 2, True, 21)
    out = q3attn.paged_decode_fp8(q.to(cuda_device), *pool, lens_t.to(cuda_device), table.to(cuda_device), scale)
    _check_rows(pool, table, lens_t, q, out, list(range(len(lens))), scale)
    for fp8 in (True, False):
        pool, table, lens_t, q, k, v = tree_case(cuda_device, lens, 5, 16, 2, 2, fp8, True, 22)
        mask = _tree_masks(len(lens), 5, 22)
        dev = cuda_device
        out = q3attn.paged_decode_tree(q.to(dev), k.to(dev), v.to(dev), mask.to(dev), pool[0], pool[1], lens_t.to(dev), table.to(dev),
                                       scale, pool[2], pool[3])
        want, spread = attention(q, pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens_t, table, scale, (k, v, mask))
        assert_close(out, want, spread)


def test_queries_near_the_largest_number(cuda_device):
    """Queries of magnitudes up to bf16's largest against keys that bring the scores back: Q's two e4m3 parts span them."""
    pool, table, lens, q = decode_case(cuda_device, [70, 300, 9], 16, 2, 2, True, 23)
    pool[2].fill_(10)                                          # keys of up to 448 * 2^-117
    q[0] *= 2.0 ** 113                                         # scores of about 2^113 * 2^-117 * 128^0.5 * 100
    q[1] = torch.where(q[1] > 0, 2.0 ** 113, -(2.0 ** 113)).to(torch.bfloat16)
    q[1, 0, 0] = 2.0 ** 127 * 1.9921875                        # the largest; the others are 2^-14 of it
    q[2, :, 64:] = 0
    out = q3attn.paged_decode_fp8(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), SCALE)
    rows = [0, 2]
    _check_rows(pool, table, lens, q, out, rows)
    # (row 1's head 0 has scores of 2^14 times the others': not a number to compare, but one)
    want, spread = attention(q[[1]][:, None], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens[[1]], table[[1]], SCALE)
    assert_close(out[[1]][:, 1:], want[:, 0, 1:], spread[:, 0, 1:])
    assert torch.isfinite(out).all()


def test_queries_that_are_not_finite(cuda_device):
    """A query head with NaN or infinities gives NaN, and no other head does."""
    pool, table, lens, q = decode_case(cuda_device, [70, 300, 2000], 16, 2, 4, True, 24)
    clean = q3attn.paged_decode_fp8(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), SCALE)
    q[0, 1, 5] = float("nan")
    q[1, 6, 127] = float("inf")
    q[2, 3, 64] = float("-inf")
    out = q3attn.paged_decode_fp8(q.to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), SCALE)
    for b, h in ((0, 1), (1, 6), (2, 3)):
        assert torch.isnan(out[b, h]).all()
        out[b, h] = clean[b, h]
    # (a head near one that is not finite is coded by other instructions, to the same codes)
    assert torch.equal(out, clean)


@pytest.mark.parametrize("fp8", [True, False])
def test_far_pages(cuda_device, fp8):
    """Pages whose offsets pass 32 bits in a cache of 5 GiB."""
    page, hkv = 16, 8
    pages = (5 << 30) // (page * hkv * D * (1 if fp8 else 2))
    lens = [100, 1500, 17]
    near, table, lens_t, q, k, v = tree_case(cuda_device, lens, 4, page, hkv, 2, fp8, True, 25)
    n = near[0].shape[0]
    far = torch.randperm(pages // 5, generator=torch.Generator().manual_seed(1))[:n].to(cuda_device) + 4 * (pages // 5)
    caches = []
    for c in near[:2]:
        big = torch.empty((pages, hkv, page, D), dtype=torch.uint8 if fp8 else torch.bfloat16, device=cuda_device)
        src = c.transpose(1, 2)
        big.index_copy_(0, far, src.view(torch.uint8) if fp8 else src)
        big = big.view(E4M3) if fp8 else big
        caches.append(big.transpose(1, 2))
    scales = [None, None]
    if fp8:
        scales = []
        for s in near[2:]:
            big = torch.full((pages, hkv, page), 255, dtype=torch.uint8, device=cuda_device)
            big.index_copy_(0, far, s)
            scales.append(big)
    moved = torch.where(table < 0, table, far.cpu().to(torch.int32)[table.clamp(min=0).long()])
    mask = _tree_masks(3, 4, 25)
    pool = (*near[:2], *near[2:])
    want = run_tree(cuda_device, pool, table, lens_t, q, k, v, mask)
    assert torch.equal(run_tree(cuda_device, (*caches, *scales), moved, lens_t, q, k, v, mask), want)
    if fp8:
        args = (lens_t.to(cuda_device), SCALE)
        q1 = q[:, 0].to(cuda_device)
        a = q3attn.paged_decode_fp8(q1, *near, args[0], table.to(cuda_device), SCALE)
        assert torch.equal(q3attn.paged_decode_fp8(q1, *caches, *scales, args[0], moved.to(cuda_device), SCALE), a)


@pytest.mark.parametrize("lens", [[2000, 5], list(range(0, 600, 2))])
def test_graphs_that_share_their_memory(cuda_device, lens):
    """Two graphs captured into one memory pool, whose calls' workspaces lie at the same addresses, replayed in turn."""
    pool, table, lens_t, q = decode_case(cuda_device, lens, 16, 8, 2, True, 26)
    args = [(x.to(cuda_device), *pool, lens_t.to(cuda_device), table.to(cuda_device), s) for x, s in ((q, 0.1), (-q, 0.05))]
    eager = [q3attn.paged_decode_fp8(*a).clone() for a in args]
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            q3attn.paged_decode_fp8(*args[0])                  # its result is dropped: the next call may have its memory
            outs.append(q3attn.paged_decode_fp8(*a).clone())
        graphs.append(g)
    for i in (0, 1, 1, 0, 1):
        junk = torch.randn(1 << 18, device=cuda_device)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], eager[i])
        del junk


def test_trees_on_two_streams(cuda_device):
    cases = [tree_case(cuda_device, lens, 20, 16, 2, 2, fp8, True, 27) for lens, fp8 in (([2000], True), ([40, 1500, 7], False))]
    masks = [_tree_masks(len(c[2]), 20, 28) for c in cases]
    eager = [run_tree(cuda_device, *c, m) for c, m in zip(cases, masks)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for s, c, m, g in zip(streams, cases, masks, got):
            with torch.cuda.stream(s):
                g.append(run_tree(cuda_device, *c, m))
    torch.cuda.synchronize()
    for g, e in zip(got, eager):
        assert all(torch.equal(x, e) for x in g)


def test_a_row_gets_the_same_bits_whatever_the_batch_holds(cuda_device):
    """Whole rows: a row's result does not depend on its neighbours or on its place in the order."""
    lens = [500, 3, 90, 499, 0, 260] * 20
    pool, table, lens_t, q = decode_case(cuda_device, lens, 16, 4, 2, True, 29, width=32)
    args = lambda p: (q[p].to(cuda_device), *pool, lens_t[p].to(cuda_device), table[p].to(cuda_device), SCALE)
    a = q3attn.paged_decode_fp8(*args(torch.arange(120)))
    p = torch.randperm(120, generator=torch.Generator().manual_seed(2))
    b = q3attn.paged_decode_fp8(*args(p))
    assert torch.equal(b, a[p.to(cuda_device)])


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("late", [2.0, 7.0])
def test_values_near_the_largest_number(cuda_device, fp8, late):
    """One key of a value near bf16's largest, whose score is over all those before it: its probability's share is a number, and
    so is everything on the way to it.  (Keys 0 to 31 and 128 to 159 are one wave's steps.)"""
    page, n, at = 16, 170, 140
    k, v = torch.zeros((n, 1, D)), torch.zeros((n, 1, D))
    k[at, 0, 0], v[at, 0, ::2], v[at, 0, 1::2] = 1.0, 3e38, -3e38
    k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, 176 - n)).to(torch.bfloat16).to(cuda_device) for x in (k, v))
    slots = torch.arange(176, device=cuda_device)
    if fp8:
        pool = q3attn.fp8_cache(11, page, 1)
        q3attn.paged_write_fp8(k, v, slots, *pool)
    else:
        pool = (k.view(11, page, 1, D), v.view(11, page, 1, D), None, None)
    table, lens = torch.arange(11, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
    q = torch.zeros((1, 1, 2, D), dtype=torch.bfloat16)
    q[..., 0] = late * 128 ** 0.5
    own = torch.zeros((1, 1, 1, D), dtype=torch.bfloat16)
    mask = torch.zeros((1, 1, 1), dtype=torch.bool)
    want, spread = attention(q, pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, SCALE, (own, own, mask))
    assert torch.isfinite(want).all()
    assert_close(run_tree(cuda_device, pool, table, lens, q, own, own, mask), want, spread)
    if fp8:
        out = q3attn.paged_decode_fp8(q[:, 0].to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), SCALE)
        assert_close(out, want[:, 0], spread[:, 0])


@pytest.mark.parametrize("fp8", [True, False])
def test_long_rows_whose_query_rows_fill_the_chip(cuda_device, fp8):
    """64 nodes of 256 heads over 16 KV heads: 512 workgroups a row, so its steps stay together however long it is."""
    pool, table, lens, q, k, v = tree_case(cuda_device, [1500], 64, 16, 16, 16, fp8, True, 30, width=4096)
    mask = _tree_masks(1, 64, 31)
    out = run_tree(cuda_device, pool, table, lens, q, k, v, mask)
    nodes = [0, 31, 63]
    want, spread = attention(q[:, nodes], pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, SCALE,
                             (k, v, mask[:, nodes]))
    assert_close(out[:, nodes], want, spread)
