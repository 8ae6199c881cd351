"""CPU tests of the 4-bit pool's and the page moves' boundary: what the C entry points refuse before any launch, and that the Python ops
refuse CPU tensors."""
import ctypes

import pytest
import torch

import q3attn
from fp4_reference import pool_values
from q3attn import _lib

POOL = dict(kc=16, vc=16, sp=8192, st=64, sh=1024, ks=16, vs=16, ssp=512, ssh=64, pages=8, page=16)


def _err():
    return _lib.lib().q3a_last_error().decode()


def _pool(a):
    return (a["kc"], a["vc"], a["sp"], a["st"], a["sh"], a["ks"], a["vs"], a["ssp"], a["ssh"], a["pages"], a["page"])


ROWS = dict(POOL, k=16, k_st=1024, k_sh=128, v=16, v_st=1024, v_sh=128, slots=16, T=4, Hkv=8, D=128)


def _write(**kw):
    a = dict(ROWS, **kw)
    return _lib.lib().q3a_paged_write_fp4(a["k"], a["k_st"], a["k_sh"], a["v"], a["v_st"], a["v_sh"], a["slots"], *_pool(a), a["T"], a["Hkv"],
                                          a["D"], None)


def _read(**kw):
    a = dict(ROWS, **kw)
    return _lib.lib().q3a_paged_read_fp4(*_pool(a), a["slots"], a["k"], a["k_st"], a["k_sh"], a["v"], a["v_st"], a["v_sh"], a["T"], a["Hkv"],
                                         a["D"], None)


ATT = dict(POOL, q=16, q_sb=2048, q_sh=128, kn=16, kn_sb=1024, kn_sh=128, vn=16, vn_sb=1024, vn_sh=128, lens=16, bt=16, bt_sb=4, max_pages=4,
           out=16, o_sb=2048, o_sh=128, ws=16, ws_bytes=1 << 30, B=2, Hq=16, Hkv=8, D=128, scale=0.088)


def _decode(append, **kw):
    a = dict(ATT, **kw)
    new = (a["kn"], a["kn_sb"], a["kn_sh"], a["vn"], a["vn_sb"], a["vn_sh"]) if append else ()
    f = _lib.lib().q3a_paged_decode_fp4_append if append else _lib.lib().q3a_paged_decode_fp4
    return f(a["q"], a["q_sb"], a["q_sh"], *new, *_pool(a), a["lens"], a["bt"], a["bt_sb"], a["max_pages"], a["out"], a["o_sb"], a["o_sh"],
             a["ws"], a["ws_bytes"], a["B"], a["Hq"], a["Hkv"], a["D"], a["scale"], None)


POOL_BAD = [(dict(kc=None), "null"), (dict(vs=None), "null"), (dict(page=24), "page_size"), (dict(page=0), "page_size"),
            (dict(page=8), "page_size"), (dict(kc=24), "aligned"), (dict(st=48), "stride"), (dict(st=72), "aligned"),
            (dict(sh=-64), "stride"), (dict(sp=8), "aligned"), (dict(ssp=2), "scale"), (dict(ssh=-4), "scale"), (dict(ks=18), "scale"),
            (dict(st=1 << 27), "stride"), (dict(pages=-1), "num_pages"), (dict(Hkv=0), ""), (dict(D=64), "head_dim")]


@pytest.mark.parametrize("kw,frag", POOL_BAD + [(dict(k=None), "null"), (dict(slots=None), "null"), (dict(v=24), "aligned"),
                                                (dict(k_st=1028), "aligned"), (dict(T=-1), "token count"), (dict(T=1 << 40), "token"),
                                                (dict(slots=20), "aligned"), (dict(page=1 << 27), "page_size")])
def test_write_and_read_refuse(kw, frag):
    for f in (_write, _read):
        assert f(**kw) == -22 and frag in _err()


@pytest.mark.parametrize("kw,frag", POOL_BAD + [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(lens=None), "null"), (dict(bt=None), "null"), (dict(q=20), "aligned"),
    (dict(q_sh=132), "aligned"), (dict(o_sb=2049), "aligned"), (dict(Hq=12), "query heads"), (dict(Hq=8 * 17), "query heads"),
    (dict(Hq=65, Hkv=65), "query heads"), (dict(B=-1), "batch"), (dict(B=65536), "batch"), (dict(max_pages=-1), "table"),
    (dict(max_pages=1 << 27), "table"), (dict(sp=1 << 36), "64 GiB")])
def test_decode_refuses(kw, frag):
    for append in (False, True):
        assert _decode(append, **kw) == -22 and frag in _err()


@pytest.mark.parametrize("kw,frag", [(dict(kn=None), "null"), (dict(vn=8), "aligned"), (dict(kn_sb=1028), "aligned")])
def test_new_rows_refused(kw, frag):
    assert _decode(True, **kw) == -22 and frag in _err()


def test_workspace_and_empty_calls():
    need = _lib.lib().q3a_paged_decode_tree_workspace_bytes(2, 1, 16, 8, 128, 4096, 16)
    assert need > 0
    for append in (False, True):
        assert _decode(append, max_pages=4096, ws_bytes=need - 1) == -28 and "workspace" in _err()
        assert _decode(append, max_pages=4096, ws=None) == -28
        assert _decode(append, B=0) == 0
    assert _write(T=0, k=None, v=None, slots=None) == 0 and _read(T=0) == 0


def _cache(**kw):
    a = dict(base=256, stride_page=2048, stride_1=0, stride_0=0, n_1=1, n_0=1, run_bytes=2048, num_pages=8)
    a.update(kw)
    return _lib.PageCache(*(a[n] for n, _ in _lib.PageCache._fields_))


def _copy(caches, pairs=3, src=16, dst=16):
    arr = (_lib.PageCache * max(1, len(caches)))(*caches)
    return _lib.lib().q3a_paged_copy(arr, len(caches), src, dst, pairs, None)


@pytest.mark.parametrize("kw,frag", [(dict(base=None), "null"), (dict(base=18), "multiples of 4"), (dict(run_bytes=0), "positive"),
                                     (dict(run_bytes=6), "multiples of 4"), (dict(n_0=0), "positive"), (dict(stride_page=-4), "strides"),
                                     (dict(stride_page=2), "multiples of 4"), (dict(n_0=2, stride_0=6), "multiples of 4"),
                                     (dict(n_1=2, stride_1=-8), "strides"), (dict(num_pages=-1), "positive"), (dict(run_bytes=1 << 33), "8 GiB"),
                                     (dict(run_bytes=1 << 31, n_0=2), "8 GiB")])
def test_copy_refuses(kw, frag):
    assert _copy([_cache(), _cache(**kw)]) == -22 and frag in _err() and "cache 1" in _err()


def test_copy_refuses_lists():
    assert _copy([_cache()], pairs=-1) == -22 and "pairs" in _err()
    assert _copy([_cache()], src=None) == -22 and "null" in _err()
    assert _lib.lib().q3a_paged_copy(None, 1, 16, 16, 1, None) == -22 and "list" in _err()
    assert _copy([], pairs=4) == 0 and _copy([_cache()], pairs=0, src=None, dst=None) == 0


def _compact(**kw):
    a = dict(caches=[16, 32], scales=[1, 2], row=64, blocks=4, sp=8192, st=64, sh=1024, ssp=512, ssh=64, pages=8, page=16, keep=1, keep_sb=64,
             width=64, lens=16, bt=16, bt_sb=4, max_pages=4, new=16, B=2, Hkv=8)
    a.update(kw)
    ptrs = [None if x is None else (ctypes.c_void_p * max(1, len(x)))(*x) for x in (a["caches"], a["scales"])]
    return _lib.lib().q3a_paged_compact(*ptrs, 0 if a["caches"] is None else len(a["caches"]), a["row"], a["blocks"], a["sp"], a["st"], a["sh"],
                                        a["ssp"], a["ssh"], a["pages"], a["page"], a["keep"], a["keep_sb"], a["width"], a["lens"], a["bt"],
                                        a["bt_sb"], a["max_pages"], a["new"], a["B"], a["Hkv"], None)


@pytest.mark.parametrize("kw,frag", [
    (dict(caches=None), "at least one"), (dict(caches=[]), "at least one"), (dict(caches=[16, None]), "cache 1"), (dict(caches=[16, 24]), "cache 1"),
    (dict(scales=None), "null scales"), (dict(scales=[1, None]), "cache 1"), (dict(row=96), "rows of"), (dict(row=256, blocks=1), "rows of"),
    (dict(row=128, blocks=4), "rows of"), (dict(B=-1), "batch"), (dict(B=65536), "batch"), (dict(Hkv=0), "heads"), (dict(Hkv=65537), "heads"),
    (dict(page=24), "page_size"), (dict(page=0), "page_size"), (dict(pages=-1), "num_pages"), (dict(max_pages=1 << 25), "table"),
    (dict(max_pages=-1), "table"), (dict(width=-1), "width"), (dict(sp=8), "strides"), (dict(st=48), "stride"), (dict(sh=-16), "strides"),
    (dict(ssp=-1), "strides"), (dict(lens=None), "null"), (dict(new=None), "null"), (dict(keep=None), "null"), (dict(bt=None), "null")])
def test_compact_refuses(kw, frag):
    assert _compact(**kw) == -22 and frag in _err()


def test_compact_of_no_rows():
    assert _compact(B=0, lens=None, new=None) == 0


def test_cpu_tensors_raise():
    pool = q3attn.fp4_cache(2, device="cpu")
    x, q = torch.zeros((1, 8, 128), dtype=torch.bfloat16), torch.zeros((1, 16, 128), dtype=torch.bfloat16)
    n, bt = torch.zeros((1,), dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32)
    slot = torch.zeros((1,), dtype=torch.int64)
    keep = torch.ones((1, 4), dtype=torch.bool)
    for call in (lambda: q3attn.paged_write_fp4(x, x, slot, *pool), lambda: q3attn.paged_read_fp4(*pool, slot),
                 lambda: q3attn.paged_decode_fp4(q, *pool, n, bt, 1.0), lambda: q3attn.paged_decode_fp4_append(q, x, x, *pool, n, bt, 1.0),
                 lambda: q3attn.paged_copy(list(pool), n, n), lambda: q3attn.paged_compact(pool[:2], keep, n, bt, pool[2:]),
                 lambda: q3attn.paged_copy([], n, n)):
        with pytest.raises(RuntimeError):
            call()


def test_fp4_cache_layout():
    kc, vc, ks, vs = q3attn.fp4_cache(3, 32, 4, device="cpu")
    assert kc.shape == (3, 32, 4, 64) and kc.stride() == vc.stride() == (32 * 4 * 64, 64, 32 * 64, 1)
    assert ks.shape == vs.shape == (3, 4, 4, 32) and kc.dtype == ks.dtype == torch.uint8
    assert not pool_values(kc, ks).any()
