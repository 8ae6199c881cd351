"""Copies of pages and compaction of rows against the same moves in numpy: contents are compared byte for byte, over whole pools."""
import numpy as np
import pytest
import torch

import q3attn
from fp8_reference import table_for

pytestmark = pytest.mark.gpu


def _bytes(t):
    return t.cpu().contiguous().view(torch.uint8)


def _random(shape, seed, dev):
    return torch.randint(0, 256, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.uint8).to(dev)


def _want_copy(caches, src, dst):
    want = []
    for c in caches:
        w = _bytes(c).clone()
        for p, q in zip(src, dst):
            if 0 <= p < len(w) and 0 <= q < len(w):
                w[q] = _bytes(c)[p]
        want.append(w)
    return want


def _check_copy(caches, src, dst):
    want = _want_copy(caches, src, dst)
    ids = [torch.tensor(x, dtype=torch.int32, device=caches[0].device) for x in (src, dst)]
    q3attn.paged_copy(caches, *ids)
    for i, (c, w) in enumerate(zip(caches, want)):
        assert torch.equal(_bytes(c), w), i


def test_copy_of_all_pools(cuda_device):
    """bf16, 8-bit and 4-bit layers with their scales in one list, a page forked thrice, pairs that are left out."""
    bf16 = [_random((20, 16, 8, 256), i, cuda_device).view(torch.bfloat16) for i in range(4)]
    fp8 = [t for _ in range(2) for t in q3attn.fp8_cache(20, device=cuda_device)]
    fp4 = [t for _ in range(2) for t in q3attn.fp4_cache(20, device=cuda_device)]
    for i, t in enumerate(fp8 + fp4):
        t.view(torch.uint8).copy_(_random(t.shape, 50 + i, cuda_device))
    _check_copy(bf16 + fp8 + fp4, [3, 3, 3, 0, -1, 20, 5, 7, 11], [4, 19, 1, 2, 6, 8, -2, 7, 1 << 30])


@pytest.mark.parametrize("pairs", [1, 2, 65, 700])
@pytest.mark.parametrize("shape", [(16, 8, 128), (48, 3, 64), (4,), (16, 1, 4)])
def test_copy_sizes(cuda_device, shape, pairs):
    pages = 2 * pairs + 3
    ids = np.random.default_rng(pairs).permutation(pages)
    caches = [_random((pages, *shape), i, cuda_device) for i in range(3)]
    _check_copy(caches, ids[:pairs].tolist(), ids[pairs:2 * pairs].tolist())


def test_copy_of_pages_in_pieces(cuda_device):
    """Views whose pages are not one run: K and V interleaved, some of the heads, heads first, rows with gaps."""
    both = _random((9, 2, 16, 4, 64), 1, cuda_device)
    gaps = _random((9, 16, 4, 72), 2, cuda_device)
    heads = _random((9, 4, 16, 64), 3, cuda_device).transpose(1, 2)
    rest = [both.clone(), gaps.clone(), heads.clone()]
    caches = [both[:, 0], both[:, 1], gaps[..., :64], gaps[:, :, 1:3, :8], heads[:, :, 1:3], heads]
    src, dst = [0, 8, 3], [1, 2, 7]
    _check_copy(caches[:2], src, dst)
    assert torch.equal(both[[0, 3, 4, 5, 6, 8]], rest[0][[0, 3, 4, 5, 6, 8]])
    _check_copy(caches[2:3], src, dst)
    assert torch.equal(gaps[..., 64:], rest[1][..., 64:])
    gaps.copy_(rest[1])
    _check_copy(caches[3:4], src, dst)
    untouched = torch.ones_like(gaps, dtype=torch.bool)
    untouched[:, :, 1:3, :8] = False
    assert torch.equal(gaps[untouched], rest[1][untouched])
    _check_copy(caches[4:5], src, dst)
    assert torch.equal(heads[:, :, [0, 3]], rest[2][:, :, [0, 3]])
    _check_copy(caches[5:6], src, dst)
    _check_copy([both[:, 0], heads, both[:, 1], gaps[..., :64]], [4], [5])


def test_copy_of_many_caches_and_shapes(cuda_device):
    """More caches than a launch takes, and more shapes."""
    caches = [_random((5, 16 * (1 + i // 40)), i, cuda_device) for i in range(300)]
    _check_copy(caches, [0, 4], [2, 3])
    caches = [_random((5 + i % 7, 16, 2 + i % 7, 64), i, cuda_device) for i in range(40)]
    _check_copy(caches, [0, 4, 9], [2, 3, 8])


def test_copy_far_pages(cuda_device):
    pages = 600_000
    cache = torch.empty((pages, 16, 8, 64), dtype=torch.uint8, device=cuda_device)
    assert cache.numel() > 1 << 32
    cache[[5, pages - 1]] = _random((2, 16, 8, 64), 1, cuda_device)
    q3attn.paged_copy([cache], *(torch.tensor(x, dtype=torch.int32, device=cuda_device) for x in ([5, pages - 1], [pages - 2, 6])))
    assert torch.equal(cache[pages - 2], cache[5]) and torch.equal(cache[6], cache[pages - 1])


def test_copy_captured_and_replayed(cuda_device):
    caches = [_random((30, 16, 8, 128), i, cuda_device) for i in range(8)]
    src, dst = (torch.zeros(6, dtype=torch.int32, device=cuda_device) for _ in range(2))
    dst.fill_(-1)
    q3attn.paged_copy(caches, src, dst)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q3attn.paged_copy(caches, src, dst)
    for seed in range(3):
        ids = np.random.default_rng(seed).permutation(30)
        want = _want_copy(caches, ids[:6].tolist(), ids[6:12].tolist())
        src.copy_(torch.from_numpy(ids[:6].astype(np.int32)))
        dst.copy_(torch.from_numpy(ids[6:12].astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        for c, w in zip(caches, want):
            assert torch.equal(_bytes(c), w)


def test_copy_refusals(cuda_device):
    c = torch.zeros((4, 16, 8, 64), dtype=torch.uint8, device=cuda_device)
    ids = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    q3attn.paged_copy([c], ids[:0], ids[:0])
    q3attn.paged_copy([c[:0], c], ids, ids)
    bad = [([], ids, ids), ([c], ids.long(), ids.long()), ([c], ids, ids[:1]), ([c], ids.cpu(), ids), ([c, c.cpu()], ids, ids),
           ([torch.zeros((4, 3), dtype=torch.uint8, device=cuda_device)], ids, ids), ([c[:, :, :, ::2]], ids, ids),
           ([torch.zeros((4, 1, 8, 64), dtype=torch.uint8, device=cuda_device).expand(4, 16, 8, 64)], ids, ids),
           ([c], ids.view(1, 2), ids.view(1, 2)), ([torch.zeros((4, 4, 4, 4, 8), device=cuda_device)[:, ::2, ::2, ::2, ::2]], ids, ids)]
    for args in bad:
        with pytest.raises(RuntimeError, match="q3a|q3attn"):
            q3attn.paged_copy(*args)


# ---------------------------------------------------------------------------------------------------- compaction

def _pools(kind, layers, pages, page, hkv, head_major, seed, dev):
    """(caches, scales) of ``layers`` layers' K and V with random bytes."""
    row = {"bf16": 256, "fp8": 128, "fp4": 64}[kind]
    caches, scales = [], []
    for i in range(2 * layers):
        t = _random((pages, hkv, page, row) if head_major else (pages, page, hkv, row), seed + i, dev)
        t = t.transpose(1, 2) if head_major else t
        caches.append(t if kind == "fp4" else t.view(torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn))
        if kind != "bf16":
            scales.append(_random((pages, hkv, page) if kind == "fp8" else (pages, hkv, 4, page), 99 + seed + i, dev))
    return caches, scales


def _want_compact(caches, scales, keep, lens, table, page):
    """The caches' and scales' bytes after the moves, and the new lengths."""
    caches, scales = [_bytes(t).clone().numpy() for t in caches], [_bytes(t).clone().numpy() for t in scales]
    pages, new = caches[0].shape[0], []
    for b, n in enumerate(lens):
        n = min(int(n), table.shape[1] * page)
        if n <= 0:
            new.append(n)
            continue
        kept = [t for t in range(n) if t >= keep.shape[1] or keep[b, t]]
        new.append(len(kept))
        for t, d in ((t, d) for d, t in enumerate(kept) if t != d):
            p, q = int(table[b, t // page]), int(table[b, d // page])
            if not (0 <= p < pages and 0 <= q < pages):
                continue
            for c in caches:
                c[q, d % page] = c[p, t % page]
            for s in scales:
                s[q, ..., d % page] = s[p, ..., t % page]
    return caches, scales, new


def _check_compact(caches, scales, keep, lens, table, page):
    dev = caches[0].device
    want = _want_compact(caches, scales, keep.numpy(), lens, table.numpy(), page)
    seqlens = torch.tensor(list(lens), dtype=torch.int32, device=dev)
    got = q3attn.paged_compact(caches, keep.to(dev), seqlens, table.to(dev), scales)
    assert got.dtype == torch.int32 and got.tolist() == want[2]
    assert seqlens.tolist() == list(lens)
    for t, w in zip(list(caches) + list(scales), want[0] + want[1]):
        assert torch.equal(_bytes(t), torch.from_numpy(w))
    return got


@pytest.mark.parametrize("kind,page,hkv,head_major", [("bf16", 16, 8, False), ("bf16", 48, 1, True), ("fp8", 16, 2, True), ("fp8", 64, 3, False),
                                                      ("fp4", 16, 8, True), ("fp4", 256, 2, False)])
def test_compact_ragged_rows(cuda_device, kind, page, hkv, head_major):
    lens = [0, 1, 2, 15, 16, 17, 33, 64, 100, 129, 300, -4, 47]
    used = sum(-(-max(n, 0) // page) for n in lens)
    caches, scales = _pools(kind, 2, used + 2, page, hkv, head_major, page, cuda_device)
    table = table_for(lens, page, used + 2, -(-max(lens) // page), page)
    keep = torch.rand((len(lens), max(lens)), generator=torch.Generator().manual_seed(page)) < torch.linspace(0.1, 0.95, len(lens))[:, None]
    _check_compact(caches, scales, keep, lens, table, page)


@pytest.mark.parametrize("pattern", ["all", "none", "first", "last", "second half", "alternate", "window", "all but the first", "all but the last"])
def test_compact_patterns(cuda_device, pattern):
    """Long rows, whose masks take several spans of the kernel, with lengths at a span's border."""
    lens = [2048, 2049, 4096, 5001, 2047]
    t, n = torch.arange(5001)[None], torch.tensor(lens)[:, None]
    keep = {"all": t >= 0, "none": t < 0, "first": t == 0, "last": t == n - 1, "second half": t >= n // 2, "alternate": t % 2 == 1,
            "window": (t < 4) | (t >= n - 700), "all but the first": t > 0, "all but the last": t != n - 1}[pattern].expand(5, -1).contiguous()
    used = sum(-(-x // 16) for x in lens)
    caches, scales = _pools("fp4", 1, used + 1, 16, 1, True, 3, cuda_device)
    _check_compact(caches, scales, keep, lens, table_for(lens, 16, used + 1, -(-5001 // 16), 3), 16)


def test_compact_mask_narrower_and_wider_than_rows(cuda_device):
    lens = [100, 40, 7]
    for width in (0, 1, 30, 100, 150):
        caches, scales = _pools("bf16", 1, 14, 16, 2, False, width, cuda_device)
        keep = torch.rand((3, width), generator=torch.Generator().manual_seed(width)) < 0.5
        _check_compact(caches, scales, keep, lens, table_for(lens, 16, 14, 7, 1), 16)
    wide = torch.rand((3, 160), generator=torch.Generator().manual_seed(5)) < 0.5
    caches, scales = _pools("fp8", 1, 14, 16, 2, True, 8, cuda_device)
    table, dev = table_for(lens, 16, 14, 7, 1), cuda_device
    want = _want_compact(caches, scales, wide[:, 3:].numpy(), lens, table.numpy(), 16)
    got = q3attn.paged_compact(caches, wide.to(dev)[:, 3:], torch.tensor(lens, dtype=torch.int32, device=dev), table.to(dev), scales)
    assert got.tolist() == want[2] and torch.equal(_bytes(caches[1]), torch.from_numpy(want[0][1]))


def test_compact_pages_missing_and_rows_past_the_table(cuda_device):
    lens = [100, 200, 64]
    caches, scales = _pools("fp4", 1, 20, 16, 2, True, 4, cuda_device)
    table = table_for([100, 64, 64], 16, 20, 7, 2)
    table[0, 2], table[2, 0], table[1, 3] = -1, 20, 1 << 30
    keep = torch.rand((3, 200), generator=torch.Generator().manual_seed(6)) < 0.6
    _check_compact(caches, scales, keep, lens, table[:, :7], 16)


def test_compact_many_caches_and_rows(cuda_device):
    caches, scales = _pools("fp8", 70, 30, 16, 1, True, 5, cuda_device)      # more caches than a launch takes
    lens = [70, 33, 200]
    keep = torch.rand((3, 200), generator=torch.Generator().manual_seed(7)) < 0.5
    _check_compact(caches, scales, keep, lens, table_for(lens, 16, 30, 13, 3), 16)
    lens = np.random.default_rng(1).integers(-1, 60, 400).tolist()
    used = sum(-(-max(n, 0) // 16) for n in lens)
    caches, scales = _pools("fp4", 1, used, 16, 2, False, 6, cuda_device)
    keep = torch.rand((400, 60), generator=torch.Generator().manual_seed(8)) < 0.7
    _check_compact(caches, scales, keep, lens, table_for(lens, 16, used, 4, 4), 16)


def test_compact_far_pages(cuda_device):
    pages, dev = 600_000, cuda_device
    cache = torch.empty((pages, 16, 8, 64), dtype=torch.uint8, device=dev)
    scale = torch.empty((pages, 8, 4, 16), dtype=torch.uint8, device=dev)
    table = torch.tensor([[3, pages - 1, pages - 2]], dtype=torch.int32, device=dev)
    cache[table[0].long()] = _random((3, 16, 8, 64), 1, dev)
    scale[table[0].long()] = _random((3, 8, 4, 16), 2, dev)
    rows, exps = cache[table[0].long()].view(48, 8, 64), scale[table[0].long()].permute(0, 3, 1, 2).reshape(48, 8, 4)
    keep = torch.arange(48, device=dev)[None] % 3 != 1
    n = q3attn.paged_compact([cache], keep, torch.tensor([48], dtype=torch.int32, device=dev), table, [scale])
    assert n.tolist() == [32]
    assert torch.equal(cache[table[0].long()].view(48, 8, 64)[:32], rows[keep[0]])
    assert torch.equal(scale[table[0].long()].permute(0, 3, 1, 2).reshape(48, 8, 4)[:32], exps[keep[0]])


def test_compact_captured_and_replayed(cuda_device):
    dev, lens = cuda_device, [90, 300, 17]
    caches, scales = _pools("fp8", 2, 40, 16, 2, True, 9, dev)
    table = table_for(lens, 16, 40, 19, 5)
    keep = torch.ones((3, 300), dtype=torch.bool, device=dev)
    seqlens, bt = torch.tensor(lens, dtype=torch.int32, device=dev), table.to(dev)
    q3attn.paged_compact(caches, keep, seqlens, bt, scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = q3attn.paged_compact(caches, keep, seqlens, bt, scales)
    for seed in range(3):
        mask = torch.rand((3, 300), generator=torch.Generator().manual_seed(seed)) < 0.6
        now = [n - 5 * seed for n in lens]
        want = _want_compact(caches, scales, mask.numpy(), now, table.numpy(), 16)
        keep.copy_(mask)
        seqlens.copy_(torch.tensor(now))
        graph.replay()
        torch.cuda.synchronize()
        assert new.tolist() == want[2]
        for t, w in zip(caches + scales, want[0] + want[1]):
            assert torch.equal(_bytes(t), torch.from_numpy(w))


def test_compact_refusals(cuda_device):
    dev = cuda_device
    caches, scales = _pools("fp4", 1, 4, 16, 2, True, 1, dev)
    lens, table = torch.tensor([20], dtype=torch.int32, device=dev), torch.zeros((1, 2), dtype=torch.int32, device=dev)
    keep = torch.ones((1, 20), dtype=torch.bool, device=dev)
    assert q3attn.paged_compact(caches, keep[:0], lens[:0], table[:0], scales).shape == (0,)
    bf = [torch.zeros((4, 16, 2, 128), dtype=torch.bfloat16, device=dev)]
    bad = [([], keep, lens, table, []), (caches, keep, lens, table, []), (caches, keep, lens, table, scales[:1]), (bf, keep, lens, table, scales[:1]),
           (caches, keep.int(), lens, table, scales), (caches, keep[0], lens, table, scales), (caches, keep, lens.long(), table, scales),
           (caches, keep, lens, table.long(), scales), (caches, keep.cpu(), lens, table, scales), (caches, keep, lens, table[:, :, None], scales),
           ([caches[0], caches[1].contiguous()], keep, lens, table, scales), (caches, keep, lens, table, [scales[0], scales[1][..., :8]]),
           (caches, keep, lens, table, [s.transpose(2, 3).contiguous().transpose(2, 3) for s in scales]), ([bf[0].half()], keep, lens, table, []),
           ([bf[0][..., :64]], keep, lens, table, []), ([bf[0][:0]], keep, lens, table, []), (caches, torch.cat([keep, keep]), lens, table, scales),
           (caches, keep.expand(1, 20).as_strided((1, 10), (20, 2)), lens, table, scales)]
    for args in bad:
        with pytest.raises(RuntimeError, match="q3a|q3attn"):
            q3attn.paged_compact(*args)


def test_copy_and_compact_compiled(cuda_device):
    """Inside torch.compile: both write the caller's pools."""
    dev = cuda_device
    caches = [_random((8, 16, 2, 256), i, dev).view(torch.bfloat16) for i in range(2)]
    src, dst = (torch.tensor([x], dtype=torch.int32, device=dev) for x in (1, 5))
    keep = torch.arange(40, device=dev)[None] % 2 == 0
    lens, table = torch.tensor([40], dtype=torch.int32, device=dev), torch.tensor([[5, 2, 3]], dtype=torch.int32, device=dev)
    want = [c.clone() for c in caches]

    def step(a, b, keep):
        q3attn.paged_copy([a, b], src, dst)
        return q3attn.paged_compact([a, b], keep | (keep ^ keep), lens, table) + 1

    n = step(*want, keep)
    got = torch.compile(step, dynamic=False)(*caches, keep)
    assert torch.equal(n, got) and n.tolist() == [21]
    for a, b in zip(caches, want):
        assert torch.equal(_bytes(a), _bytes(b))
