"""How precisely decode over the 8-bit pool and attention for trees compute: probabilities are held to 16 bits in the product with V,
infinities in a bf16 pool's values included."""
import pytest
import torch

import q3attn
from fp8_reference import D, E4M3, attention, pool_values, table_for
from q3attn import _lib
from test_gpu_decode_tree import _tree_masks

pytestmark = pytest.mark.gpu

SCALE = D ** -0.5
LENS = [2, 3, 5, 8, 33, 40, 170, 600]


def _pool(lens, hkv, fp8, dev, seed, value=None):
    """A bf16 or 8-bit pool of unit-variance rows (values all ``value`` where it is given) and its table."""
    used = sum(-(-n // 16) for n in lens)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((used * 16, hkv, D), generator=g).to(torch.bfloat16) for _ in range(2))
    if value is not None:
        v = value.expand_as(v).contiguous()
    k, v = k.to(dev), v.to(dev)
    if fp8:
        pool = q3attn.fp8_cache(used, 16, hkv, device=dev)
        q3attn.paged_write_fp8(k, v, torch.arange(used * 16, device=dev), *pool)
    else:
        pool = (k.view(used, 16, hkv, D), v.view(used, 16, hkv, D), None, None)
    return pool, table_for(lens, 16, used, -(-max(lens) // 16), seed)


def _tree(dev, pool, table, lens, q, k, v, mask):
    return q3attn.paged_decode_tree(q.to(dev), k.to(dev), v.to(dev), mask.to(dev), pool[0], pool[1], lens.to(dev), table.to(dev), SCALE,
                                    pool[2], pool[3])


def _assert_precise(got, want, spread):
    """Half a bf16 step of the result (2^-8 of it); of the spread 2^-15 for the two parts of a probability (the first leaves 2^-7
    of it at worst, the second 2^-8 of that) and 2^-13 for the scores: 128 products of at most 4 in all, each rounded once or
    cut off: 128 * 2^-23 * 4 = 2^-14, and exp2, sums and quotients of 2^-23 each."""
    got = got.cpu().double()
    off = (got - want).abs() - 2.0 ** -8 * want.abs() - (2.0 ** -15 + 2.0 ** -13) * spread
    assert not (off > 1e-30).any(), float((off / spread.clamp(min=1e-30)).max())


@pytest.mark.parametrize("nodes,hkv,group", [(1, 4, 2), (5, 2, 2), (20, 2, 2), (40, 1, 1)])
@pytest.mark.parametrize("fp8", [True, False])
def test_probabilities_in_the_product(cuda_device, fp8, nodes, hkv, group):
    g = torch.Generator().manual_seed(nodes)
    lens = torch.tensor(LENS, dtype=torch.int32)
    pool, table = _pool(LENS, hkv, fp8, cuda_device, nodes)
    # scores of unit-variance keys: sum |q_d k_d| * scale is about 128 * 0.2 * 0.64 * 128^-0.5 = 1.4
    q = (0.2 * torch.randn((len(LENS), nodes, hkv * group, D), generator=g)).to(torch.bfloat16)
    k, v = (torch.randn((len(LENS), nodes, hkv, D), generator=g).to(torch.bfloat16) for _ in range(2))
    mask = _tree_masks(len(LENS), nodes, nodes)
    vals = pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3])
    want, spread = attention(q, *vals, lens, table, SCALE, (k, v, mask))
    _assert_precise(_tree(cuda_device, pool, table, lens, q, k, v, mask), want, spread)
    if fp8:
        q1 = q[:, 0].to(cuda_device)
        out = q3attn.paged_decode_fp8(q1, *pool, lens.to(cuda_device), table.to(cuda_device), SCALE)
        want, spread = attention(q[:, :1], *vals, lens, table, SCALE)
        _assert_precise(out, want[:, 0], spread[:, 0])


@pytest.mark.parametrize("fp8", [True, False])
def test_equal_values_come_back(cuda_device, fp8):
    """Whatever the scores, the mean of values that are all the same is that value: what the probabilities' two parts and fp32
    sums leave (2^-15 and 2^-20 of it) is under half a bf16 step (2^-9 of it at least), so it comes back bit for bit."""
    g = torch.Generator().manual_seed(1)
    value = torch.randn((1, 1, D), generator=g).to(torch.bfloat16)
    if fp8:
        value = value.float().to(E4M3).to(torch.bfloat16)      # held as it is
    lens = torch.tensor(LENS, dtype=torch.int32)
    pool, table = _pool(LENS, 2, fp8, cuda_device, 2, value)
    q = torch.randn((len(LENS), 6, 4, D), generator=g).to(torch.bfloat16)
    k = torch.randn((len(LENS), 6, 2, D), generator=g).to(torch.bfloat16)
    v = value.expand_as(k).contiguous()
    out = _tree(cuda_device, pool, table, lens, q, k, v, _tree_masks(len(LENS), 6, 3)).cpu()
    assert torch.equal(out, value.expand_as(out))
    if fp8:
        out = q3attn.paged_decode_fp8(q[:, 0].to(cuda_device), *pool, lens.to(cuda_device), table.to(cuda_device), SCALE).cpu()
        assert torch.equal(out, value.expand_as(out))


@pytest.mark.parametrize("nodes", [3, 20])
def test_infinite_cached_values(cuda_device, nodes):
    """An infinity among a bf16 pool's values reaches every node as that infinity, also where its key's probability is a power of
    two (the row's largest: its second part would round to 0) or far below the others' (2^-90)."""
    lens = torch.tensor([70], dtype=torch.int32)
    pool, table = _pool([70], 1, False, cuda_device, 4)
    k = pool[0].view(-1, D)
    slot = [int(table[0, t // 16]) * 16 + t % 16 for t in range(70)]
    k[slot] = 0
    k[slot[10], 0] = 1.0
    k[slot[40], 0] = -2.0
    v = pool[1].view(-1, D)
    v[slot[10], 3], v[slot[40], 5], v[slot[50], 7], v[slot[50], 9], v[slot[51], 9] = (
        float("inf"), float("-inf"), float("inf"), float("inf"), float("-inf"))
    q = torch.zeros((1, nodes, 2, D), dtype=torch.bfloat16)
    q[..., 0] = 256.0                                          # scores of 22.6, 0 and -45.3: 2^-33 and 2^-98 of the largest
    own = torch.zeros((1, nodes, 1, D), dtype=torch.bfloat16)
    mask = torch.eye(nodes, dtype=torch.bool)[None]
    out = _tree(cuda_device, pool, table, lens, q, own, own, mask).cpu().float()
    inf = torch.full_like(out[..., 0], float("inf"))
    assert torch.equal(out[..., 3], inf) and torch.equal(out[..., 5], -inf) and torch.equal(out[..., 7], inf)
    assert torch.isnan(out[..., 9]).all()
    rest = [d for d in range(D) if d not in (3, 5, 7, 9)]
    assert torch.isfinite(out[..., rest]).all()


@pytest.mark.parametrize("large", [2.0 ** 12, 2.0 ** 17, 2.0 ** 24, 3.0e38])
@pytest.mark.parametrize("nodes,hkv,group", [(1, 2, 2), (3, 1, 4), (30, 1, 2)])
def test_small_query_elements_beside_large_ones(cuda_device, nodes, hkv, group, large):
    """Queries whose first element is far larger than the others, over keys that are 0 there: the others are the score.  Only some
    heads have it, and one has elements of every size."""
    g = torch.Generator().manual_seed(nodes)
    lens = torch.tensor(LENS, dtype=torch.int32)
    used = sum(-(-n // 16) for n in LENS)
    kv = torch.randn((2, used * 16, hkv, D), generator=g).to(torch.bfloat16)
    kv[0, ..., 0] = 0
    pool = q3attn.fp8_cache(used, 16, hkv, device=cuda_device)
    q3attn.paged_write_fp8(kv[0].to(cuda_device), kv[1].to(cuda_device), torch.arange(used * 16, device=cuda_device), *pool)
    table = table_for(LENS, 16, used, -(-max(LENS) // 16), nodes)
    q = (0.2 * torch.randn((len(LENS), nodes, hkv * group, D), generator=g)).to(torch.bfloat16)
    q[:, ::2, 0, 0] = large
    q[1::2, :, -1, 0] = -large
    q[2, 0, -1] *= torch.exp2(-torch.arange(D) / 4.0).to(torch.bfloat16)
    k, v = (torch.randn((len(LENS), nodes, hkv, D), generator=g).to(torch.bfloat16) for _ in range(2))
    k[..., 0] = 0
    mask = _tree_masks(len(LENS), nodes, nodes)
    vals = pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3])
    want, spread = attention(q, *vals, lens, table, SCALE, (k, v, mask))
    _assert_precise(_tree(cuda_device, pool, table, lens, q, k, v, mask), want, spread)
    want, spread = attention(q[:, :1], *vals, lens, table, SCALE)
    args = lens.to(cuda_device), table.to(cuda_device), SCALE
    _assert_precise(q3attn.paged_decode_fp8(q[:, 0].to(cuda_device), *pool, *args), want[:, 0], spread[:, 0])
    now = torch.tensor([n - 1 for n in LENS], dtype=torch.int32)    # the last token again, as the step's own
    last = [int(table[b, (n - 1) // 16]) * 16 + (n - 1) % 16 for b, n in enumerate(LENS)]
    out = q3attn.paged_decode_fp8_append(q[:, 0].to(cuda_device), kv[0, last].to(cuda_device), kv[1, last].to(cuda_device), *pool,
                                         now.to(cuda_device), *args[1:])
    _assert_precise(out, want[:, 0], spread[:, 0])


@pytest.mark.parametrize("nodes,hkv,group", [(1, 2, 2), (3, 1, 4), (30, 1, 2)])
def test_small_query_elements_in_chunks(cuda_device, nodes, hkv, group):
    """The same in a table so wide that rows are cut into chunks; a head that is not finite beside it gives NaN, and no other does."""
    g = torch.Generator().manual_seed(nodes)
    lens, width = torch.tensor([2500, 3, 0, 1100], dtype=torch.int32), 4096
    used = 157 + 1 + 69
    kv = torch.randn((2, used * 16, hkv, D), generator=g).to(torch.bfloat16)
    kv[0, ..., 0] = 0
    pool = q3attn.fp8_cache(used, 16, hkv, device=cuda_device)
    q3attn.paged_write_fp8(kv[0].to(cuda_device), kv[1].to(cuda_device), torch.arange(used * 16, device=cuda_device), *pool)
    table = table_for(lens.tolist(), 16, used, width, nodes)
    assert _lib.lib().q3a_paged_decode_tree_workspace_bytes(4, nodes, hkv * group, hkv, D, width, 16) > 0
    q = (0.2 * torch.randn((4, nodes, hkv * group, D), generator=g)).to(torch.bfloat16)
    q[:, ::2, 0, 0] = 2.0 ** 20
    k, v = (torch.randn((4, nodes, hkv, D), generator=g).to(torch.bfloat16) for _ in range(2))
    k[..., 0] = 0
    mask = _tree_masks(4, nodes, nodes)
    bad = q.clone()
    bad[0, 0, 1, 5], bad[3, -1, -1, 9] = float("inf"), float("nan")
    vals = pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3])
    args = lens.to(cuda_device), table.to(cuda_device), SCALE
    for n, own in ((nodes, (k, v, mask)), (1, None)):
        want, spread = attention(q[:, :n], *vals, lens, table, SCALE, own)
        for qq in (q, bad):
            if own is not None:
                out = _tree(cuda_device, pool, table, lens, qq, k, v, mask)
            else:
                out = q3attn.paged_decode_fp8(qq[:, 0].to(cuda_device), *pool, *args)[:, None]
            if qq is bad:
                lost = ~torch.isfinite(qq[:, :n].float()).all(-1)
                assert torch.isnan(out[lost.to(cuda_device)]).all() and int(lost.sum()) == (2 if n == nodes else 1 + (nodes == 1))
                out = torch.where(lost[..., None].to(cuda_device), want.to(cuda_device).to(torch.bfloat16), out)
            _assert_precise(out, want, spread)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("nodes", [5, 40])
def test_probabilities_in_chunks(cuda_device, fp8, nodes):
    g = torch.Generator().manual_seed(nodes)
    lens = [2500, 3, 0, 1100]
    pool, table = _pool(lens, 2, fp8, cuda_device, nodes)
    assert _lib.lib().q3a_paged_decode_tree_workspace_bytes(4, nodes, 4, 2, D, table.shape[1], 16) > 0
    q = (0.2 * torch.randn((4, nodes, 4, D), generator=g)).to(torch.bfloat16)
    k, v = (torch.randn((4, nodes, 2, D), generator=g).to(torch.bfloat16) for _ in range(2))
    mask = _tree_masks(4, nodes, nodes)
    lens = torch.tensor(lens, dtype=torch.int32)
    want, spread = attention(q, pool_values(pool[0], pool[2]), pool_values(pool[1], pool[3]), lens, table, SCALE, (k, v, mask))
    _assert_precise(_tree(cuda_device, pool, table, lens, q, k, v, mask), want, spread)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("nodes", [3, 20])
def test_infinite_queries_give_nan(cuda_device, fp8, nodes):
    """Also where every score is -inf (exp(-inf - -inf)), over cached and own keys; other heads and nodes as without."""
    lens = torch.tensor([1, 40, 0], dtype=torch.int32)
    pool, table = _pool([1, 40, 1], 1, fp8, cuda_device, 5)
    if not fp8:
        pool[0].copy_(pool[0].abs())
    g = torch.Generator().manual_seed(6)
    q = (0.2 * torch.randn((3, nodes, 2, D), generator=g)).to(torch.bfloat16)
    k, v = (torch.randn((3, nodes, 1, D), generator=g).to(torch.bfloat16) for _ in range(2))
    k = k.abs()
    mask = _tree_masks(3, nodes, nodes)
    bad = q.clone()
    for b, n, h, value in ((0, 0, 1, "-inf"), (1, nodes - 1, 0, "-inf"), (2, 1, 0, "-inf"), (2, 2, 1, "inf")):
        bad[b, n, h, 7] = float(value)
    lost = torch.isinf(bad).any(-1)
    out = _tree(cuda_device, pool, table, lens, bad, k, v, mask).cpu()
    clean = _tree(cuda_device, pool, table, lens, q, k, v, mask).cpu()
    assert torch.isnan(out[lost]).all() and torch.equal(out[~lost], clean[~lost])
