"""Decode over the 8-bit pool and attention for trees inside torch.compile, where their fake implementations stand for them."""
import pytest
import torch

import q3attn
from test_gpu_decode_tree import _case, _tree_masks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("transposed", [True, False])
def test_compiled_attention(cuda_device, fp8, transposed):
    """One graph without breaks, equal to the eager step; q may lie in another order than its shape's, the result does not."""
    dev = cuda_device
    pool, table, lens, q, k, v = _case(dev, [70, 5, 900], 4, 16, 2, 2, fp8, True, 1)
    mask, table, lens = _tree_masks(3, 4, 1).to(dev), table.to(dev), lens.to(dev)
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    if transposed:
        q = q.transpose(1, 2).contiguous().transpose(1, 2)

    def step(q, k, v, *pool):
        o = q3attn.paged_decode_tree(q * 2, k, v, mask, pool[0], pool[1], lens, table, 0.1, pool[2], pool[3])
        one = q3attn.paged_decode_fp8(q[:, 0] * 2, *pool, lens, table, 0.1) if fp8 else o[:, 0]
        return o.view(3, 4, -1) + 1, one.view(3, -1) * 2

    with torch.no_grad():
        want = step(q, k, v, *pool)
        got = torch.compile(step, dynamic=False, fullgraph=True)(q, k, v, *pool)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and a.stride() == b.stride()
