"""The 4-bit pool's write and read against their definition in 64 bits.  Scales are powers of two, so codes, exponent bytes and values
read back are compared exactly."""
import pytest
import torch

import q3attn
from fp4_reference import pack, quantise, values

pytestmark = pytest.mark.gpu


def _pool(pages, page, hkv, layout, dev, fill=0x55):
    """A pool whose bytes are all ``fill``, in the layout of fp4_cache, token-major, or with gaps between rows."""
    if layout == "head":
        pool = q3attn.fp4_cache(pages, page, hkv, device=dev)
        for t in pool:
            t.fill_(fill)
        return pool
    gap = 0 if layout == "token" else 16
    caches = [torch.full((pages, page, hkv, 64 + gap), fill, dtype=torch.uint8, device=dev)[..., :64] for _ in range(2)]
    scales = [torch.full((pages, hkv + 1, 4, page), fill, dtype=torch.uint8, device=dev)[:, :hkv] for _ in range(2)]
    return (*caches, *scales)


def _special_rows(x):
    """Rows where the format can go wrong, put over the first rows of x [T, H, 128]."""
    f = x.view(-1, 128)
    rows = [
        torch.zeros(128), torch.full((128,), -0.0),
        torch.tensor([7.0, 0.25, -0.75, 1.25, -1.75, 2.5, 3.5, -5.0] * 16), torch.tensor([7.03125, 0.25, 0.5, -1.5, 3.0, 5.0, 7.0, 6.5] * 16),
        torch.tensor(([1.75 * 2.0 ** -20] + [2.0 ** -30] * 31 + [1.7578125 * 2.0 ** -20] + [2.0 ** -22] * 31) * 2),
        torch.tensor([3.38953139e38] + [1.0] * 31 + [7.0 * 2.0 ** 125] + [2.0 ** 123] * 31 + [6.0 * 2.0 ** 125] * 32 + [-2.0 ** 127] * 32),
        torch.tensor([2.0 ** -126] * 32 + [2.0 ** -127] * 32 + [1.5 * 2.0 ** -127] * 32 + [7.0 * 2.0 ** -125, 2.0 ** -133] * 16),
        torch.tensor([1.0 + i / 128 for i in range(128)]),
        torch.tensor([-(256.0 + 2 * i) for i in range(64)] + [2.0 ** -i for i in range(64)]),
        torch.tensor([float("inf")] + [1.5] * 127), torch.tensor([float("nan")] * 128),
        torch.tensor([float("-inf"), float("nan")] + [-0.0, 5.0] * 63),
    ]
    n = min(len(rows), f.shape[0])
    f[:n] = torch.stack(rows[:n]).to(torch.bfloat16)
    return x


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
        slots[[1, T - 1]] = torch.tensor([-1, pages * page])     # not written
    pool = _pool(pages, page, hkv, layout, cuda_device)
    want = [t.cpu().clone() for t in pool]
    kv = torch.cat([k, v], 1).to(cuda_device)                    # k and v as views of one tensor
    q3attn.paged_write_fp4(kv[:, :hkv], kv[:, hkv:], slots.to(cuda_device), *pool)
    for x, cache, scale in ((k, want[0], want[2]), (v, want[1], want[3])):
        code, byte = quantise(x)
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                cache[s // page, s % page] = pack(code[t])
                scale[s // page, :, :, s % page] = byte[t].to(torch.uint8)
    for got, w in zip(pool, want):
        assert torch.equal(got.cpu(), w)


@pytest.mark.parametrize("T,hkv,page,layout", [(1, 8, 16, "head"), (77, 8, 256, "token"), (35, 3, 48, "gap"), (2, 1, 16, "head")])
def test_read_gives_the_values(cuda_device, T, hkv, page, layout):
    """Any codes, at every exponent byte that the writer makes."""
    g = torch.Generator().manual_seed(T)
    pages = -(-T // page) + 2
    pool = _pool(pages, page, hkv, layout, cuda_device)
    for t in pool[:2]:
        t.copy_(torch.randint(0, 256, t.shape, generator=g).to(torch.uint8))
    for t in pool[2:]:
        t.copy_(torch.randint(2, 253, t.shape, generator=g).to(torch.uint8))
    pool[2][0] = 255
    slots = torch.randint(0, pages * page, (T,), generator=g)
    if T > 3:
        slots[[0, 3]] = torch.tensor([-5, pages * page])
        slots[1:3] = torch.tensor([page - 1, 0])
    got = q3attn.paged_read_fp4(*pool, slots.to(cuda_device))
    live = (slots >= 0) & (slots < pages * page)
    at = torch.where(live, slots, 0)
    for x, cache, scale in zip(got, pool[:2], pool[2:]):
        want = values(cache.cpu()[at // page, at % page], scale.cpu()[at // page, :, :, at % page])
        want[~live] = 0
        assert x.dtype == torch.bfloat16
        assert torch.equal(torch.nan_to_num(x.cpu().double(), 5.5e38, 6e38), torch.nan_to_num(want, 5.5e38, 6e38))


def test_written_rows_come_back(cuda_device):
    """Write and read many tokens: the values of the codes, and no more than half a step off."""
    T, hkv = 5000, 8
    g = torch.Generator(device=cuda_device).manual_seed(1)
    k, v = (torch.randn((T, hkv, 128), generator=g, device=cuda_device).to(torch.bfloat16) for _ in range(2))
    pool = q3attn.fp4_cache(400, 16, hkv, device=cuda_device)
    slots = torch.randperm(6400, device=cuda_device)[:T]
    q3attn.paged_write_fp4(k, v, slots, *pool)
    for x, got in zip((k, v), q3attn.paged_read_fp4(*pool, slots)):
        code, byte = quantise(x.cpu())
        assert torch.equal(got.cpu().double(), values(pack(code), byte))


def test_captured_and_replayed(cuda_device):
    pool = q3attn.fp4_cache(10, 16, 8, device=cuda_device)
    k = torch.randn((50, 8, 128), device=cuda_device).to(torch.bfloat16)
    slots = torch.arange(50, device=cuda_device)
    q3attn.paged_write_fp4(k, k, slots, *pool)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q3attn.paged_write_fp4(k, k, slots, *pool)
        out = q3attn.paged_read_fp4(*pool, slots)
    for seed in range(3):
        k.copy_(torch.randn((50, 8, 128), generator=torch.Generator().manual_seed(seed)))
        slots.copy_(torch.randperm(160, generator=torch.Generator().manual_seed(seed))[:50])
        graph.replay()
        torch.cuda.synchronize()
        code, byte = quantise(k.cpu())
        for x in out:
            assert torch.equal(x.cpu().double(), values(pack(code), byte))


def test_nothing_to_do_and_refusals(cuda_device):
    pool = q3attn.fp4_cache(4, 16, 8, device=cuda_device)
    k = torch.zeros((3, 8, 128), dtype=torch.bfloat16, device=cuda_device)
    slots = torch.arange(3, device=cuda_device)
    q3attn.paged_write_fp4(k[:0], k[:0], slots[:0], *pool)
    assert q3attn.paged_read_fp4(*pool, slots[:0])[0].shape == (0, 8, 128)
    bad = [(k.float(), k, slots, *pool), (k, k[:, :4], slots, *pool), (k, k, slots.int(), *pool), (k, k, slots[:2], *pool),
           (k, k, slots.cpu(), *pool), (k[..., ::2], k[..., ::2], slots, *pool), (k, k, slots, pool[0].view(torch.int8), *pool[1:]),
           (k, k, slots, *pool[:2], pool[2][..., :8], pool[3][..., :8]), (k, k, slots, pool[0][:2], *pool[1:]),
           (torch.zeros((3, 8, 136), dtype=torch.bfloat16, device=cuda_device)[..., 1:129], k, slots, *pool)]
    for args in bad:
        with pytest.raises(RuntimeError, match="q3a|q3attn"):
            q3attn.paged_write_fp4(*args)
    odd = torch.zeros((4, 16, 8, 72), dtype=torch.uint8, device=cuda_device)[..., :64]
    for args in [(odd, odd, *pool[2:], slots), (pool[0].half(), pool[1].half(), *pool[2:], slots), (*pool, slots.int())]:
        with pytest.raises(RuntimeError, match="q3a|q3attn"):
            q3attn.paged_read_fp4(*args)
