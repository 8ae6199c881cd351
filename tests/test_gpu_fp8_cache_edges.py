"""The 8-bit pool and trees at edges of their arguments: pools of 2^31 slots and more, tables without a page."""
import pytest
import torch

import q3attn
from fp8_reference import D, E4M3, assert_close, attention, quantise
from test_gpu_decode_tree import _tree_masks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages", [(1 << 27) - 1, 1 << 27, (1 << 27) + 5])
def test_slots_past_32_bits(cuda_device, pages):
    """All pages are one page of memory (page stride 0): a slot's place in its page is what counts."""
    page, hkv = 16, 2
    caches = [torch.zeros((1, page, hkv, D), dtype=torch.uint8, device=cuda_device).view(E4M3) for _ in range(2)]
    scales = [torch.full((1, hkv, page), 127, dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    pool = [c.expand(pages, *c.shape[1:]) for c in caches + scales]
    x = torch.randn((6, hkv, D), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    last = pages * page
    slots = torch.tensor([0, 16 * 1000 + 3, last - 1, last, last + 5, 1 << 62], device=cuda_device)
    q3attn.paged_write_fp8(x.to(cuda_device), -x.to(cuda_device), slots, *pool)
    code, s = quantise(x)
    want = (code * torch.exp2((s - 127).double())[..., None])
    k, v = q3attn.paged_read_fp8(*pool, slots)
    assert torch.equal(k[:3].cpu().double(), want[:3]) and torch.equal(v[:3].cpu().double(), -want[:3])
    assert not k[3:].any() and not v[3:].any()
    rest = [o for o in range(page) if o not in (0, 3, 15)]
    assert not caches[0].view(torch.uint8)[:, rest].any() and (scales[0][..., rest] == 127).all()


@pytest.mark.parametrize("fp8", [True, False])
def test_table_without_a_page(cuda_device, fp8):
    """Rows have no cached tokens, whatever their lengths say; a tree attends its own keys, an append has no room."""
    dev, B, N = cuda_device, 3, 4
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn((B, N, h, D), generator=g).to(torch.bfloat16) for h in (4, 2, 2))
    lens = torch.tensor([0, 7, -1], dtype=torch.int32)
    table = torch.empty((B, 0), dtype=torch.int32)
    pool = q3attn.fp8_cache(2, 16, 2, device=dev)
    bf16 = [torch.zeros((2, 16, 2, D), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    kc, vc, ks, vs = pool if fp8 else (*bf16, None, None)
    mask = _tree_masks(B, N, 3)
    out = q3attn.paged_decode_tree(q.to(dev), k.to(dev), v.to(dev), mask.to(dev), kc, vc, lens.to(dev), table.to(dev), 0.1, ks, vs)
    none = torch.zeros((2, 16, 2, D), dtype=torch.float64)
    want, spread = attention(q, none, none, [0, 0, -1], table, 0.1, (k, v, mask))
    assert_close(out, want, spread)
    if fp8:
        before = [t.view(torch.uint8).clone() for t in pool]
        assert not q3attn.paged_decode_fp8(q[:, 0].to(dev), *pool, lens.to(dev), table.to(dev), 0.1).any()
        assert not q3attn.paged_decode_fp8_append(q[:, 0].to(dev), k[:, 0].to(dev), v[:, 0].to(dev), *pool, lens.to(dev), table.to(dev), 0.1).any()
        assert all(torch.equal(a.view(torch.uint8), b) for a, b in zip(pool, before))
