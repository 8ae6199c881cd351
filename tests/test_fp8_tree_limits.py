"""CPU tests of the sizes that the 8-bit pool's and the tree attention's C entry points refuse before any launch."""
import pytest

from q3attn import _lib
from test_fp8_tree_capi import _decode, _err, _read, _tree, _write


@pytest.mark.parametrize("kw", [dict(pages=(1 << 22) + 1), dict(pages=2, sp=1 << 36), dict(pages=1 << 20, sp=1 << 45),
                                dict(pages=1 << 20, ssp=1 << 20), dict(pages=1 << 20, ssp=1 << 50)])
def test_attention_refuses_caches_past_its_offsets(kw):
    assert _decode(False, **kw) == -22 and "64 GiB" in _err()
    assert _decode(True, **kw) == -22 and "64 GiB" in _err()
    assert _tree(**kw) == -22 and "64 GiB" in _err()


def test_a_bf16_cache_counts_two_bytes_an_element():
    bf16 = dict(ks=None, vs=None, ssp=0, ssh=0)
    assert _tree(pages=(1 << 21) + 1, **bf16) == -22 and "64 GiB" in _err()


@pytest.mark.parametrize("max_pages,page", [((1 << 24) + 1, 16), (1 << 20, 512)])
def test_attention_refuses_tables_past_its_counts(max_pages, page):
    kw = dict(max_pages=max_pages, page=page)
    assert _decode(False, **kw) == -22 and "2^28" in _err()
    assert _tree(**kw) == -22 and "2^28" in _err()
    assert _lib.lib().q3a_paged_decode_tree_workspace_bytes(2, 5, 16, 8, 128, max_pages, page) == 0


def test_write_and_read_refuse_head_counts():
    for f in (_write, _read):
        assert f(Hkv=65537, T=1) == -22 and "65536" in _err()


@pytest.mark.parametrize("batch,heads,tokens", [(1, 8, 16384), (1024, 1, 1 << 20), (64, 8, 32768), (7, 64, 1 << 28)])
def test_workspace_is_bounded(batch, heads, tokens):
    """Chunks are as many as the compute units hold, and one a row more: at most 512 (or a row each) of 16 query rows a head."""
    need = _lib.lib().q3a_paged_decode_tree_workspace_bytes(batch, 1, heads, heads, 128, tokens // 16, 16)
    assert need <= 8 * batch + 16 + (512 + batch * heads) * 16 * 130 * 4


def test_no_workspace_where_one_rows_query_rows_fill_the_chip():
    for batch, nodes, hq, hkv in ((1, 256, 1024, 64), (3, 64, 256, 16), (1024, 256, 1024, 64)):
        assert _lib.lib().q3a_paged_decode_tree_workspace_bytes(batch, nodes, hq, hkv, 128, 1 << 20, 16) == 0
