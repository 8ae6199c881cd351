"""CPU tests of the workspace of decode over the 8-bit pool and of tree attention across shapes: as the header says, it does not grow with
the batch, so a buffer sized for the largest one is refused where a smaller one needs more."""
from q3attn import _lib
from test_fp8_tree_capi import _decode, _err, _tree


def _bytes(batch, nodes=1, hq=16, hkv=8, tokens=2048):
    return _lib.lib().q3a_paged_decode_tree_workspace_bytes(batch, nodes, hq, hkv, 128, tokens // 16, 16)


def test_a_smaller_call_may_need_more():
    assert _bytes(576) < _bytes(1)
    assert _bytes(1, nodes=64) > _bytes(1, nodes=8) and _bytes(64, nodes=256) < _bytes(1, nodes=64)
    assert _bytes(24, tokens=512) < _bytes(24)


def test_a_buffer_of_the_largest_batch_is_refused_for_a_smaller_one():
    shape = dict(N=1, max_pages=128)
    assert _decode(False, B=1, **shape, ws=None, ws_bytes=_bytes(576)) == -28 and str(_bytes(1)) in _err()
    assert _decode(True, B=1, **shape, ws_bytes=_bytes(1) - 1) == -28
    assert _tree(B=1, N=8, max_pages=128, ws_bytes=_bytes(576, nodes=8)) == -28
