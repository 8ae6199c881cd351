"""CPU tests of the 8-bit pool's and the tree attention's boundary: what the C entry points refuse before any launch, that the
Python ops refuse CPU tensors, and pins of the reference the GPU tests compare with."""
import pytest
import torch

import q3attn
from fp8_reference import E4M3, attention, pool_values, quantise
from q3attn import _lib

POOL = dict(kc=16, vc=16, sp=16384, st=128, sh=2048, ks=16, vs=16, ssp=128, ssh=16, pages=8, page=16)


def _err():
    return _lib.lib().q3a_last_error().decode()


def _write(**kw):
    a = dict(POOL, k=16, k_st=1024, k_sh=128, v=16, v_st=1024, v_sh=128, slots=16, T=4, Hkv=8, D=128)
    a.update(kw)
    return _lib.lib().q3a_paged_write_fp8(a["k"], a["k_st"], a["k_sh"], a["v"], a["v_st"], a["v_sh"], a["slots"], a["kc"], a["vc"],
                                          a["sp"], a["st"], a["sh"], a["ks"], a["vs"], a["ssp"], a["ssh"], a["pages"], a["page"],
                                          a["T"], a["Hkv"], a["D"], None)


def _read(**kw):
    a = dict(POOL, k=16, k_st=1024, k_sh=128, v=16, v_st=1024, v_sh=128, slots=16, T=4, Hkv=8, D=128)
    a.update(kw)
    return _lib.lib().q3a_paged_read_fp8(a["kc"], a["vc"], a["sp"], a["st"], a["sh"], a["ks"], a["vs"], a["ssp"], a["ssh"],
                                         a["pages"], a["page"], a["slots"], a["k"], a["k_st"], a["k_sh"], a["v"], a["v_st"],
                                         a["v_sh"], a["T"], a["Hkv"], a["D"], None)


ATT = dict(POOL, q=16, q_sb=2048, q_sn=2048, q_sh=128, kn=16, kn_sb=1024, kn_sn=1024, kn_sh=128, vn=16, vn_sb=1024, vn_sn=1024,
           vn_sh=128, mask=None, m_sb=0, m_sn=0, lens=16, bt=16, bt_sb=4, max_pages=4, out=16, o_sb=2048, o_sn=2048, o_sh=128, ws=16,
           ws_bytes=1 << 30, B=2, N=5, Hq=16, Hkv=8, D=128, scale=0.088)


def _decode(append, **kw):
    a = dict(ATT)
    a.update(kw)
    new = (a["kn"], a["kn_sb"], a["kn_sh"], a["vn"], a["vn_sb"], a["vn_sh"]) if append else ()
    f = _lib.lib().q3a_paged_decode_fp8_append if append else _lib.lib().q3a_paged_decode_fp8
    return f(a["q"], a["q_sb"], a["q_sh"], *new, a["kc"], a["vc"], a["sp"], a["st"], a["sh"], a["ks"], a["vs"], a["ssp"], a["ssh"],
             a["pages"], a["page"], a["lens"], a["bt"], a["bt_sb"], a["max_pages"], a["out"], a["o_sb"], a["o_sh"], a["ws"],
             a["ws_bytes"], a["B"], a["Hq"], a["Hkv"], a["D"], a["scale"], None)


def _tree(**kw):
    a = dict(ATT)
    a.update(kw)
    return _lib.lib().q3a_paged_decode_tree(
        a["q"], a["q_sb"], a["q_sn"], a["q_sh"], a["kn"], a["kn_sb"], a["kn_sn"], a["kn_sh"], a["vn"], a["vn_sb"], a["vn_sn"],
        a["vn_sh"], a["mask"], a["m_sb"], a["m_sn"], a["kc"], a["vc"], a["sp"], a["st"], a["sh"], a["ks"], a["vs"], a["ssp"],
        a["ssh"], a["pages"], a["page"], a["lens"], a["bt"], a["bt_sb"], a["max_pages"], a["out"], a["o_sb"], a["o_sn"], a["o_sh"],
        a["ws"], a["ws_bytes"], a["B"], a["N"], a["Hq"], a["Hkv"], a["D"], a["scale"], None)


POOL_BAD = [(dict(kc=None), "null"), (dict(vs=None), "null"), (dict(page=24), "page_size"), (dict(page=0), "page_size"),
            (dict(page=8), "page_size"), (dict(kc=24), "aligned"), (dict(st=120), "stride"), (dict(st=136), "aligned"),
            (dict(sh=-128), "stride"), (dict(sp=8), "aligned"), (dict(ssp=2), "scale"), (dict(ssh=-4), "scale"), (dict(ks=18), "scale"),
            (dict(st=1 << 27), "stride"), (dict(pages=-1), "num_pages"), (dict(Hkv=0), ""), (dict(D=64), "head_dim")]


@pytest.mark.parametrize("kw,frag", POOL_BAD + [(dict(k=None), "null"), (dict(slots=None), "null"), (dict(v=24), "aligned"),
                                                (dict(k_st=1028), "aligned"), (dict(T=-1), "token count"), (dict(T=1 << 40), "token"),
                                                (dict(slots=20), "aligned")])
def test_write_and_read_refuse(kw, frag):
    for f in (_write, _read):
        assert f(**kw) == -22 and frag in _err()


@pytest.mark.parametrize("kw,frag", POOL_BAD + [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(lens=None), "null"), (dict(bt=None), "null"), (dict(q=20), "aligned"),
    (dict(q_sh=132), "aligned"), (dict(o_sb=2049), "aligned"), (dict(Hq=12), "query heads"), (dict(Hq=8 * 17), "query heads"),
    (dict(Hq=65, Hkv=65), "query heads"), (dict(B=-1), "batch"), (dict(B=65536), "batch"), (dict(max_pages=-1), "table"),
    (dict(max_pages=1 << 27), "table")])
def test_decode_and_tree_refuse(kw, frag):
    for f in (lambda **k: _decode(False, **k), lambda **k: _decode(True, **k), _tree):
        assert f(**kw) == -22 and frag in _err()


@pytest.mark.parametrize("kw,frag", [(dict(kn=None), "null"), (dict(vn=8), "aligned"), (dict(kn_sb=1028), "aligned")])
def test_new_rows_refused(kw, frag):
    for f in (lambda **k: _decode(True, **k), _tree):
        assert f(**kw) == -22 and frag in _err()


@pytest.mark.parametrize("kw,frag", [(dict(N=0), "query tokens"), (dict(N=257), "query tokens"), (dict(ks=None), "null"),
                                     (dict(ks=None, vs=None, st=100), "stride"), (dict(ks=None, vs=None, kc=8), "aligned")])
def test_tree_refuses(kw, frag):
    assert _tree(**kw) == -22 and frag in _err()


def test_workspace():
    L = _lib.lib()
    need = L.q3a_paged_decode_tree_workspace_bytes(2, 5, 16, 8, 128, 4096, 16)
    assert need > 0
    assert _tree(max_pages=4096, ws_bytes=need - 1) == -28 and "workspace" in _err()
    assert _tree(max_pages=4096, ws=None) == -28
    assert _tree(max_pages=4096, ws=8) == -28
    assert L.q3a_paged_decode_tree_workspace_bytes(2, 5, 16, 8, 128, 1, 16) == 0     # one chunk
    assert L.q3a_paged_decode_tree_workspace_bytes(0, 5, 16, 8, 128, 4096, 16) == 0
    assert L.q3a_paged_decode_tree_workspace_bytes(2, 5, 15, 8, 128, 4096, 16) == 0  # a shape the calls refuse


def test_empty_calls_are_no_ops():
    assert _write(T=0, k=None, v=None, slots=None) == 0 and _read(T=0) == 0
    assert _decode(False, B=0) == 0 and _decode(True, B=0) == 0 and _tree(B=0) == 0


def test_cpu_tensors_raise():
    pool = q3attn.fp8_cache(2, device="cpu")
    x = torch.zeros((1, 8, 128), dtype=torch.bfloat16)
    q = torch.zeros((1, 16, 128), dtype=torch.bfloat16)
    n, bt = torch.zeros((1,), dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32)
    slot = torch.zeros((1,), dtype=torch.int64)
    for call in (lambda: q3attn.paged_write_fp8(x, x, slot, *pool), lambda: q3attn.paged_read_fp8(*pool, slot),
                 lambda: q3attn.paged_decode_fp8(q, *pool, n, bt, 1.0),
                 lambda: q3attn.paged_decode_fp8_append(q, x, x, *pool, n, bt, 1.0),
                 lambda: q3attn.paged_decode_tree(q[:, None], x[:, None], x[:, None], None, *pool[:2], n, bt, 1.0, *pool[2:])):
        with pytest.raises(RuntimeError):
            call()


def test_fp8_cache_layout():
    kc, vc, ks, vs = q3attn.fp8_cache(3, 32, 4, device="cpu")
    assert kc.shape == (3, 32, 4, 128) and kc.stride() == vc.stride() == (32 * 4 * 128, 128, 32 * 128, 1)
    assert ks.shape == vs.shape == (3, 4, 32) and kc.dtype == E4M3
    assert not pool_values(kc, ks).any()


def test_reference_codes_are_torchs():
    """The reference's rounding against torch's conversion, and its scale against its definition's bounds."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn((500, 128), generator=g) * torch.exp(20 * torch.randn((500, 1), generator=g))).to(torch.bfloat16)
    x = x.clamp(-1e38, 1e38)
    code, s = quantise(x)
    two = torch.pow(torch.tensor(2.0, dtype=torch.float64), (s - 127).double())[:, None]
    assert torch.equal((x.double() / two).float().to(E4M3).float().double(), code)
    top = x.double().abs().amax(1, keepdim=True)
    assert (top <= 448 * two).all() and ((top > 224 * two) | (s == 10)[:, None]).all()


def test_reference_attention_is_torchs():
    g = torch.Generator().manual_seed(1)
    q, kv = torch.randn((1, 3, 4, 128), generator=g), torch.randn((2, 40, 2, 128), generator=g, dtype=torch.float64)
    own = torch.randn((2, 1, 3, 2, 128), generator=g)
    mask = torch.tensor([[[1, 0, 0], [1, 1, 0], [0, 0, 1]]], dtype=torch.bool)
    pool = kv.view(2, 5, 8, 2, 128)
    table = torch.tensor([[3, 0, 4]], dtype=torch.int32)
    out, _ = attention(q, pool[0], pool[1], [20], table, 0.1, (own[0], own[1], mask))
    ids = torch.tensor([3] * 8 + [0] * 8 + [4] * 4) * 8 + torch.tensor(list(range(8)) * 2 + [0, 1, 2, 3])
    k = torch.cat([kv[0][ids], own[0, 0].double()]).transpose(0, 1).repeat_interleave(2, 0)
    v = torch.cat([kv[1][ids], own[1, 0].double()]).transpose(0, 1).repeat_interleave(2, 0)
    full = torch.cat([torch.ones((3, 20), dtype=torch.bool), mask[0]], 1)
    want = torch.nn.functional.scaled_dot_product_attention(q[0].double().transpose(0, 1), k, v, attn_mask=full, scale=0.1)
    assert torch.allclose(out[0].transpose(0, 1), want, rtol=1e-10, atol=1e-12)
