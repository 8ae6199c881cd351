"""The 8-bit pool's write and read against their definition in 64 bits.  Scales are powers of two, so codes, exponent bytes
and values read back are compared exactly."""
import numpy as np
import pytest
import torch

import q3attn
from fp8_reference import E4M3, quantise

pytestmark = pytest.mark.gpu


def _pool(pages, page, hkv, layout, dev, fill=0x55):
    """A pool whose bytes are all ``fill``, in the layout of fp8_cache, token-major, or with gaps between rows."""
    if layout == "head":
        pool = q3attn.fp8_cache(pages, page, hkv, device=dev)
        for t in pool:
            t.view(torch.uint8).fill_(fill)
        return pool
    gap = 0 if layout == "token" else 16
    caches = [torch.full((pages, page, hkv, 128 + gap), fill, dtype=torch.uint8, device=dev)[..., :128].view(E4M3)
              for _ in range(2)]
    scales = [torch.full((pages, hkv, page), fill, dtype=torch.uint8, device=dev) for _ in range(2)]
    return (*caches, *scales)


def _special_rows(x):
    """Rows where the format can go wrong, put over the first rows of x [T, H, 128]."""
    f = x.view(-1, 128)
    rows = [
        torch.zeros(128),
        torch.full((128,), 448.0), torch.full((128,), -448.0), torch.full((128,), 450.0),        # the scale's border
        torch.tensor([1.75 * 2.0 ** -20] + [2.0 ** -30] * 127), torch.tensor([1.7578125 * 2.0 ** -20] + [2.0 ** -30] * 127),
        torch.tensor([3.38953139e38] + [1.0] * 127),                                             # the largest bf16
        torch.tensor([2.0 ** -126] + [2.0 ** -130] * 127), torch.tensor([2.0 ** -133] * 128),    # below the least scale
        torch.tensor([2.0 ** -109] + [2.0 ** -126, 2.0 ** -127] * 63 + [0.0]),
        torch.tensor([1.0 + i / 128 for i in range(128)]),                                       # every tie of [1, 2)
        torch.tensor([-(256.0 + 2 * i) for i in range(64)] + [2.0 ** -i for i in range(64)]),
        torch.tensor([float("inf")] + [1.5] * 127), torch.tensor([float("nan")] * 128),
        torch.tensor([float("-inf"), float("nan")] + [-0.0, 5.0] * 63),
    ]
    n = min(len(rows), f.shape[0])
    f[:n] = torch.stack(rows[:n]).to(torch.bfloat16)
    return x


def _bytes(t):
    return t.cpu().contiguous().view(torch.uint8)


@pytest.mark.parametrize("T,hkv,page,layout", [(1, 8, 16, "head"), (2, 1, 16, "token"), (7, 2, 48, "gap"), (33, 8, 64, "token"),
                                               (401, 8, 16, "head"), (19, 5, 256, "head")])
def test_write_is_exact(cuda_device, T, hkv, page, layout):
    g = torch.Generator().manual_seed(T)
    k = torch.randn((T, hkv, 128), generator=g).to(torch.bfloat16)
    v = (torch.randn((T, hkv, 128), generator=g) * torch.exp(8 * torch.randn((T, hkv, 1), generator=g))).to(torch.bfloat16)
    _special_rows(k if T % 2 else v)
    pages = -(-T // page) + 3
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 3:
        slots[1], slots[3] = -1, pages * page                 # not written
    pool = _pool(pages, page, hkv, layout, cuda_device)
    kd, vd = k.to(cuda_device), v.to(cuda_device)
    wide = torch.cat([vd, vd, vd], 1)[:, hkv:2 * hkv]         # a view, as the v of a fused projection
    q3attn.paged_write_fp8(kd, wide, slots.to(cuda_device), *pool)
    torch.cuda.synchronize()
    for x, cache, scale in ((k, pool[0], pool[2]), (v, pool[1], pool[3])):
        code, s = quantise(x)
        want = torch.full((pages, page, hkv, 128), 0x55, dtype=torch.uint8)
        want_s = torch.full((pages, hkv, page), 0x55, dtype=torch.uint8)
        for t in range(T):
            if 0 <= slots[t] < pages * page:
                p, o = int(slots[t]) // page, int(slots[t]) % page
                want[p, o] = code[t].float().to(E4M3).view(torch.uint8)
                want_s[p, :, o] = s[t].to(torch.uint8)
        assert torch.equal(scale.cpu(), want_s)
        got = _bytes(cache)
        nan = want.view(E4M3).float().isnan()
        assert torch.equal(got.view(E4M3).float().isnan(), nan)
        assert torch.equal(got[~nan], want[~nan])             # -0.0 keeps its sign; every other byte too


def test_write_leaves_gaps_and_neighbours(cuda_device):
    base = torch.full((4, 16, 3, 144), 0x55, dtype=torch.uint8, device=cuda_device)
    cache = base[..., :128].view(E4M3)
    other = torch.full_like(base, 0x55)[..., :128].view(E4M3)
    scales = [torch.full((4, 3, 16), 0x55, dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    k = torch.ones((1, 3, 128), dtype=torch.bfloat16, device=cuda_device)
    q3attn.paged_write_fp8(k, k, torch.tensor([17], device=cuda_device), cache, other, *scales)
    changed = (base != 0x55).nonzero()
    assert set(map(tuple, changed[:, :2].tolist())) == {(1, 1)} and int(changed[:, 3].max()) == 127
    assert (scales[0] != 0x55).sum() == 3


def test_read_every_code(cuda_device):
    """With byte 247 the largest codes stand for more than bf16 holds (448 * 2^120 > 3.39e38; no written row has them): those
    read infinities.  Every other value is a bf16 number."""
    pool = _pool(3, 32, 2, "token", cuda_device)
    codes = torch.arange(256, dtype=torch.uint8).view(2, 128)
    for i, s in enumerate((10, 127, 247)):
        pool[0].view(torch.uint8)[i, 5] = codes.to(cuda_device)
        pool[1].view(torch.uint8)[i, 5] = codes.flip(0).to(cuda_device)
        pool[2][i, :, 5] = s
        pool[3][i, :, 5] = 257 - s if s != 127 else 127
    slots = torch.tensor([5, -1, 37, 69, 96, 1 << 40], device=cuda_device)
    k, v = q3attn.paged_read_fp8(*pool, slots)
    for i, (row, s) in enumerate(((0, 10), (2, 127), (3, 247))):
        want = (codes.view(E4M3).float().double() * 2.0 ** (s - 127)).to(torch.bfloat16).double()
        assert torch.equal(torch.nan_to_num(k[row].cpu().double(), nan=7.0), torch.nan_to_num(want, nan=7.0))
        want = codes.flip(0).view(E4M3).float().double() * 2.0 ** ((257 - s if s != 127 else 127) - 127)
        want = want.to(torch.bfloat16).double()
        assert torch.equal(torch.nan_to_num(v[row].cpu().double(), nan=7.0), torch.nan_to_num(want, nan=7.0))
    for row in (1, 4, 5):
        assert not k[row].any() and not v[row].any()


@pytest.mark.parametrize("T,hkv,page,layout", [(1, 8, 16, "head"), (130, 8, 16, "head"), (50, 3, 48, "gap")])
def test_write_then_read(cuda_device, T, hkv, page, layout):
    """What comes back is off by half an e4m3 step: 2^-4 of the value, or half of the even spacing 2^(e-9) near zero."""
    g = torch.Generator().manual_seed(T)
    x = (torch.randn((T, hkv, 128), generator=g) * 3).to(torch.bfloat16)
    y = (torch.randn((T, hkv, 128), generator=g) * torch.exp(2 * torch.randn((T, hkv, 128), generator=g))).to(torch.bfloat16)
    pool = _pool(-(-T // page) + 1, page, hkv, layout, cuda_device)
    slots = torch.randperm(T, generator=g).to(cuda_device)
    q3attn.paged_write_fp8(x.to(cuda_device), y.to(cuda_device), slots, *pool)
    k, v = q3attn.paged_read_fp8(*pool, slots)
    for a, b in ((x, k), (y, v)):
        code, s = quantise(a)
        step = torch.pow(torch.tensor(2.0, dtype=torch.float64), (s - 127).double())[..., None]
        assert torch.equal(b.cpu().double(), code * step)
        assert ((b.cpu().double() - a.double()).abs() <= torch.maximum(2.0 ** -4 * a.double().abs(), step * 2.0 ** -10)).all()


def test_far_pages(cuda_device):
    """Rows past 2^32 bytes from the pool's start."""
    pages = (1 << 32) // (16 * 8 * 128) + 8
    caches = [torch.empty((pages, 8, 16, 128), dtype=torch.uint8, device=cuda_device).view(E4M3).transpose(1, 2) for _ in range(2)]
    scales = [torch.empty((pages, 8, 16), dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    g = torch.Generator().manual_seed(1)
    x = torch.randn((40, 8, 128), generator=g).to(torch.bfloat16).to(cuda_device)
    slots = torch.cat([torch.arange(20), torch.arange(pages * 16 - 20, pages * 16)]).to(cuda_device)
    q3attn.paged_write_fp8(x, -x, slots, *caches, *scales)
    k, v = q3attn.paged_read_fp8(*caches, *scales, slots)
    code, s = quantise(x.cpu())
    want = code * torch.pow(torch.tensor(2.0, dtype=torch.float64), (s - 127).double())[..., None]
    assert torch.equal(k.cpu().double(), want) and torch.equal(v.cpu().double(), -want)


def test_pool_slots_of_a_page_pool(cuda_device):
    """PagePool's slots feed the write; its scratch seat's may repeat."""
    book = q3attn.PagePool(num_pages=12, max_seats=3, max_pages_per_seat=4, device=cuda_device)
    book.grow([0, 2], [20, 35])
    pool = q3attn.fp8_cache(12, device=cuda_device)
    seat = torch.tensor([0, 2, 2, 3, 3], device=cuda_device)
    pos = torch.tensor([19, 0, 34, 0, 0], device=cuda_device)
    x = torch.arange(5, device=cuda_device).to(torch.bfloat16).view(5, 1, 1).expand(5, 8, 128) + 1
    q3attn.paged_write_fp8(x, 2 * x, book.slot(seat, pos), *pool)
    k, v = q3attn.paged_read_fp8(*pool, book.slot(seat, pos))
    assert torch.equal(k[:3], x[:3]) and torch.equal(v[:3], 2 * x[:3])


def test_empty_calls(cuda_device):
    pool = q3attn.fp8_cache(2, device=cuda_device)
    none = torch.empty((0, 8, 128), dtype=torch.bfloat16, device=cuda_device)
    slots = torch.empty((0,), dtype=torch.int64, device=cuda_device)
    q3attn.paged_write_fp8(none, none, slots, *pool)
    k, v = q3attn.paged_read_fp8(*pool, slots)
    assert k.shape == v.shape == (0, 8, 128)


def test_refusals(cuda_device):
    pool = q3attn.fp8_cache(2, device=cuda_device)
    x = torch.zeros((3, 8, 128), dtype=torch.bfloat16, device=cuda_device)
    s = torch.zeros((3,), dtype=torch.int64, device=cuda_device)
    bad = [
        (x.float(), x, s, *pool), (x, x[:2], s, *pool), (x[:, :4], x, s, *pool), (x, x, s.int(), *pool), (x, x, s.cpu(), *pool),
        (x.transpose(0, 2).contiguous().transpose(0, 2), x, s, *pool),
        (x, x, s, pool[0].view(torch.uint8), *pool[1:]), (x, x, s, pool[0][:1], *pool[1:]), (x, x, s, *pool[:3], pool[3][:, :4]),
        (x, x, s, *pool[:2], pool[2].transpose(1, 2), pool[3].transpose(1, 2)),
        (torch.zeros((3, 8, 129), dtype=torch.bfloat16, device=cuda_device)[..., 1:], x, s, *pool),     # not 16-byte aligned
    ]
    for args in bad:
        with pytest.raises(RuntimeError, match="q3a|q3attn"):
            q3attn.paged_write_fp8(*args)
    small = q3attn.fp8_cache(2, head_dim=64, device=cuda_device)
    with pytest.raises(RuntimeError, match="head_dim"):
        q3attn.paged_read_fp8(*small, s)
    odd = q3attn.fp8_cache(2, page_size=8, device=cuda_device)
    with pytest.raises(RuntimeError, match="page_size"):
        q3attn.paged_read_fp8(*odd, s)
