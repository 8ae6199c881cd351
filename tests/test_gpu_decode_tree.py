"""Attention for trees of drafted tokens over the bf16 and the 8-bit pool against attention in 64 bits."""
import numpy as np
import pytest
import torch

import q3attn
from fp8_reference import assert_close, attention, fill_pool, pool_values, table_for

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def _tree_masks(B, N, seed):
    rng = np.random.default_rng(seed)
    m = np.zeros((B, N, N), bool)
    for b in range(B):
        for n in range(N):
            up = rng.integers(-1, n) if n else -1
            if up >= 0:
                m[b, n] = m[b, up]
            m[b, n, n] = True
    return torch.from_numpy(m)


def _case(dev, lens, N, page, hkv, group, fp8, head_major, seed, width=None):
    used = sum(-(-max(n, 0) // page) for n in lens)
    pool = fill_pool(used + 2, page, hkv, fp8, head_major, seed, dev)
    width = max(1, -(-max(lens) // page)) if width is None else width
    table = table_for(lens, page, used + 2, width, seed)
    g = torch.Generator().manual_seed(seed + 1)
    B = len(lens)
    q = torch.randn((B, N, hkv * group, 128), generator=g).to(torch.bfloat16)
    kv = torch.randn((B, N, 2 * hkv, 128), generator=g).to(torch.bfloat16)
    return pool, table, torch.tensor(lens, dtype=torch.int32), q, kv[:, :, :hkv], kv[:, :, hkv:]


def _run(dev, pool, table, lens, q, k, v, mask):
    return q3attn.paged_decode_tree(q.to(dev), k.to(dev), v.to(dev), None if mask is None else mask.to(dev), pool[0], pool[1],
                                    lens.to(dev), table.to(dev), SCALE, pool[2], pool[3])


def _full(mask, B, N):
    if mask is None:
        mask = torch.ones((N, N), dtype=torch.bool).tril()
    return mask.expand(B, N, N)


def _check(dev, pool, table, lens, q, k, v, mask):
    out = _run(dev, pool, table, lens, q, k, v, mask)
    want, spread = attention(q, pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, SCALE,
                             (k, v, _full(mask, q.shape[0], q.shape[1])))
    assert_close(out, want, spread)
    return out


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("N,hkv,group,page,head_major", [
    (1, 8, 2, 16, True), (3, 8, 2, 16, False), (8, 2, 2, 64, True), (9, 2, 2, 16, False), (16, 2, 2, 48, True),
    (17, 2, 2, 16, True), (33, 1, 2, 16, False), (64, 1, 2, 16, True), (5, 2, 16, 16, True), (70, 1, 1, 32, True),
    (11, 3, 3, 16, True)])
def test_trees(cuda_device, fp8, N, hkv, group, page, head_major):
    lens = [0, 1, 16, 33, 100, -1] if N < 40 else [0, 40, -1]
    case = _case(cuda_device, lens, N, page, hkv, group, fp8, head_major, N)
    _check(cuda_device, *case, _tree_masks(len(lens), N, N))


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("N", [1, 4, 20])
def test_chain(cuda_device, fp8, N):
    case = _case(cuda_device, [0, 7, 64, 150], N, 16, 2, 2, fp8, True, N)
    a = _check(cuda_device, *case, None)
    b = _run(cuda_device, *case, torch.ones((N, N), dtype=torch.bool).tril())       # one mask for all rows
    assert torch.equal(a, b)


@pytest.mark.parametrize("fp8", [True, False])
def test_long_contexts(cuda_device, fp8):
    case = _case(cuda_device, [3000, 1111], 6, 16, 2, 2, fp8, True, 3)
    _check(cuda_device, *case, _tree_masks(2, 6, 4))


def test_most_nodes(cuda_device):
    lens = [50]
    case = _case(cuda_device, lens, 256, 16, 1, 1, True, True, 5)
    _check(cuda_device, *case, _tree_masks(1, 256, 6))


@pytest.mark.parametrize("fp8", [True, False])
def test_empty_masks(cuda_device, fp8):
    """Nodes that see no own key: only the cache, and with an empty cache nothing (zeros)."""
    case = _case(cuda_device, [0, 20, -1], 5, 16, 2, 2, fp8, True, 7)
    mask = _tree_masks(3, 5, 7)
    mask[:, 2] = False
    out = _check(cuda_device, *case, mask)
    assert not out[0, 2].any() and out[1, 2].any() and not out[2].any()


@pytest.mark.parametrize("fp8", [True, False])
def test_masked_rows_may_hold_anything(cuda_device, fp8):
    """Padded nodes with NaN and infinite k and v, and an unpadded v with infinities that some nodes see."""
    pool, table, lens, q, k, v = _case(cuda_device, [0, 40, 7], 40, 16, 2, 2, fp8, True, 8)
    mask = _tree_masks(3, 40, 8)
    mask[:, :, 33:] = False                                   # padding: nobody sees it
    mask[:, 33:] = False
    k[:, 33:] = float("nan")
    v[:, 33:] = float("inf")
    v[1, 35] = float("nan")
    v[0, 2, 0, 5], v[0, 2, 1, 6], v[0, 20, 0, 9], v[1, 2, 1, 127] = float("inf"), float("-inf"), float("nan"), float("inf")
    k[2, 3, 0, 0] = float("nan")                               # the nodes that see node 3 get NaN, the others do not
    out = _check(cuda_device, pool, table, lens, q, k, v, mask)
    sees = mask[0, :, 2]
    assert torch.equal(torch.isinf(out[0, :, 0, 5]).cpu(), sees) and 0 < int(sees.sum()) < 40
    assert torch.equal(torch.isnan(out[2, :, 0]).any(-1).cpu(), mask[2, :, 3])


def test_strides_and_alignment(cuda_device):
    """q, k and v as views of one projection output, a mask that is a view of a wider one, a table that is one too."""
    pool, table, lens, q, k, v = _case(cuda_device, [30, 90], 7, 16, 2, 2, True, True, 9)
    qkv = torch.cat([q.reshape(2, 7, -1), k.reshape(2, 7, -1), v.reshape(2, 7, -1)], -1).to(cuda_device)
    qd, kd, vd = (x.view(2, 7, -1, 128) for x in qkv.split([4 * 128, 2 * 128, 2 * 128], -1))
    mask = _tree_masks(2, 7, 9)
    wide = torch.ones((2, 9, 13), dtype=torch.bool, device=cuda_device)
    wide[:, 1:8, 3:10] = mask.to(cuda_device)
    big = torch.full((2, table.shape[1] + 5), 1 << 30, dtype=torch.int32, device=cuda_device)
    big[:, :table.shape[1]] = table.to(cuda_device)
    out = q3attn.paged_decode_tree(qd, kd, vd, wide[:, 1:8, 3:10], pool[0], pool[1], lens.to(cuda_device),
                                   big[:, :table.shape[1]], SCALE, pool[2], pool[3])
    want, spread = attention(q, pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, SCALE, (k, v, mask))
    assert_close(out, want, spread)


@pytest.mark.parametrize("fp8", [True, False])
def test_bad_pages_and_stale_tokens(cuda_device, fp8):
    pool, table, lens, q, k, v = _case(cuda_device, [40, 21], 3, 16, 2, 2, fp8, True, 10)
    table[0, 1] = 1 << 24
    last = int(table[1, 1])
    if fp8:
        pool[1].view(torch.uint8)[last, 5:] = 0x7F
        pool[3][last, :, 5:] = 255
        pool[2][last, :, 5:] = 255
    else:
        pool[0][last, 5:] = float("nan")
        pool[1][last, 5:] = float("inf")
    _check(cuda_device, pool, table, lens, q, k, v, _tree_masks(2, 3, 10))


def test_one_node_is_decode(cuda_device):
    """N = 1 over a cache and its own key is the append form's attention, but for the new token's rounding."""
    pool, table, lens, q, k, v = _case(cuda_device, [10, 300, 31], 1, 16, 8, 2, False, False, 11, width=20)
    out = _run(cuda_device, pool, table, lens, q, k, v, None)
    kc, vc = pool[0].clone(), pool[1].clone()
    t2 = table.clone()
    for b, n in enumerate((10, 300, 31)):
        if t2[b, n // 16] < 0:
            t2[b, n // 16] = kc.shape[0] - 1 - b % 2
    ref = q3attn.paged_decode_append(q[:, 0].to(cuda_device), k[:, 0].contiguous().to(cuda_device),
                                     v[:, 0].contiguous().to(cuda_device), kc, vc, lens.to(cuda_device), t2.to(cuda_device), SCALE)
    _, spread = attention(q, pool_values(pool[0], None), pool_values(pool[1], None), lens, table, SCALE,
                          (k, v, torch.ones((3, 1, 1), dtype=torch.bool)))
    assert_close(out[:, 0], ref.cpu().double(), 2 * spread[:, 0])


def test_drafts_accepted_and_written(cuda_device):
    """The operators as a server uses them: a prompt is quantised into the pool, drafts are checked against it, the accepted
    ones are written, and the next step decodes over the result; at each step against 64 bits, the pool's rows being what the
    write of all tokens at once gives."""
    dev, B, N, hkv, hq, page = cuda_device, 3, 6, 8, 16, 16
    book = q3attn.PagePool(num_pages=64, max_seats=B, max_pages_per_seat=8, page_size=page, device=dev)
    lens = [30, 5, 63]
    book.grow(range(B), [n + N + 1 for n in lens])
    pool = q3attn.fp8_cache(64, page, hkv, device=dev)
    g = torch.Generator().manual_seed(12)
    toks = [torch.randn((n + N + 1, 2, hkv, 128), generator=g).to(torch.bfloat16) for n in lens]   # each row's k and v by position
    seat = torch.cat([torch.full((n,), b) for b, n in enumerate(lens)]).to(dev)
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev)
    prompt = torch.cat([t[:n] for t, n in zip(toks, lens)]).to(dev)
    q3attn.paged_write_fp8(prompt[:, 0], prompt[:, 1], book.slot(seat, pos), *pool)

    def check(out, q, n_rows, own):
        lens_t = torch.tensor(n_rows)
        want, spread = attention(q, pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens_t, table.cpu(), SCALE, own)
        assert_close(out, want, spread)

    table = book.block_table(torch.arange(B, device=dev))
    mask = _tree_masks(B, N, 13)
    drafts = torch.randn((B, N, 2, hkv, 128), generator=g).to(torch.bfloat16)
    path = [[0, 2], [0, 1, 4], []]                            # accepted nodes of each row
    for b, nodes in enumerate(path):
        mask[b, :, :] = torch.eye(N, dtype=torch.bool)
        for i, n in enumerate(nodes):
            mask[b, n, nodes[:i + 1]] = True
            drafts[b, n] = toks[b][lens[b] + i]
    q = torch.randn((B, N, hq, 128), generator=g).to(torch.bfloat16)
    out = q3attn.paged_decode_tree(q.to(dev), drafts[:, :, 0].to(dev), drafts[:, :, 1].to(dev), mask.to(dev), pool[0], pool[1],
                                   torch.tensor(lens, dtype=torch.int32, device=dev), table, SCALE, pool[2], pool[3])
    check(out, q, lens, (drafts[:, :, 0], drafts[:, :, 1], mask))

    slots = torch.full((B, N), -1, dtype=torch.int64)
    host = table.cpu()
    for b, nodes in enumerate(path):
        for i, n in enumerate(nodes):
            p = lens[b] + i
            slots[b, n] = int(host[b, p // page]) * page + p % page
    flat = drafts.flatten(0, 1).to(dev)
    q3attn.paged_write_fp8(flat[:, 0], flat[:, 1], slots.flatten().to(dev), *pool)
    now = [n + len(nodes) for n, nodes in zip(lens, path)]
    q1 = torch.randn((B, hq, 128), generator=g).to(torch.bfloat16)
    new = torch.stack([toks[b][n] for b, n in enumerate(now)])
    out = q3attn.paged_decode_fp8_append(q1.to(dev), new[:, 0].to(dev), new[:, 1].to(dev), *pool,
                                         torch.tensor(now, dtype=torch.int32, device=dev), table, SCALE)
    check(out[:, None], q1[:, None], [n + 1 for n in now], None)

    whole = q3attn.fp8_cache(64, page, hkv, device=dev)       # all tokens written at once
    seat = torch.cat([torch.full((n + 1,), b) for b, n in enumerate(now)]).to(dev)
    pos = torch.cat([torch.arange(n + 1) for n in now]).to(dev)
    allk = torch.cat([t[:n + 1] for t, n in zip(toks, now)]).to(dev)
    q3attn.paged_write_fp8(allk[:, 0], allk[:, 1], book.slot(seat, pos), *whole)
    for a, b in zip(q3attn.paged_read_fp8(*pool, book.slot(seat, pos)), q3attn.paged_read_fp8(*whole, book.slot(seat, pos))):
        assert torch.equal(a, b)


def test_captured_and_replayed(cuda_device):
    pool, table, lens, q, k, v = _case(cuda_device, [900, 3, 40], 5, 16, 2, 2, True, True, 14)
    args = (q.to(cuda_device), k.to(cuda_device), v.to(cuda_device), _tree_masks(3, 5, 14).to(cuda_device), pool[0], pool[1],
            lens.to(cuda_device), table.to(cuda_device), SCALE, pool[2], pool[3])
    eager = q3attn.paged_decode_tree(*args).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = q3attn.paged_decode_tree(*args)
    for _ in range(3):
        junk = torch.randn(1 << 18, device=cuda_device) * 3
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        del junk


def test_refusals(cuda_device):
    pool, table, lens, q, k, v = (x if not isinstance(x, torch.Tensor) else x.to(cuda_device)
                                  for x in _case(cuda_device, [5, 9], 4, 16, 2, 2, True, True, 1))
    mask = torch.ones((2, 4, 4), dtype=torch.bool, device=cuda_device)
    good = dict(q=q, k=k, v=v, tree_mask=mask, k_cache=pool[0], v_cache=pool[1], cache_seqlens=lens, block_table=table,
                softmax_scale=0.1, k_scale=pool[2], v_scale=pool[3])
    bad = [dict(q=q[:, :3]), dict(q=q.float()), dict(k=k[:, :, :1]), dict(v=v.half()), dict(tree_mask=mask.int()),
           dict(tree_mask=mask[:1]), dict(tree_mask=mask.transpose(1, 2)), dict(tree_mask=mask.cpu()), dict(k_scale=None),
           dict(k_scale=None, v_scale=None), dict(cache_seqlens=lens.long()), dict(block_table=table[:1]), dict(q=q.cpu()),
           dict(k=k.transpose(2, 3).contiguous().transpose(2, 3))]
    for change in bad:
        with pytest.raises(RuntimeError, match="q3a|q3attn"):
            q3attn.paged_decode_tree(**{**good, **change})
    many = torch.zeros((2, 257, 4, 128), dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(RuntimeError, match="257"):
        q3attn.paged_decode_tree(**{**good, "q": many, "k": many[:, :, :2], "v": many[:, :, :2], "tree_mask": None})
