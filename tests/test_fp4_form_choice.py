"""CPU tests of the form of launch that decode over the 4-bit pool chooses from a call's shape: chunks of rows need a workspace, whole rows
none, also where the workspace query, which knows no pool, names one.  The shapes are those of the GPU tests that are meant for one form,
so that a rule that moves does not leave a form untested."""
import pytest
import torch

from q3attn import _lib
from test_fp4_moves_capi import _decode, _err

CUS = 256                                                      # compute units: where the rule of eight waves ends


def _form(batch, hq, hkv, max_pages, page, append):
    """The call without a workspace: refused where there are chunks, else only for want of a GPU."""
    rc = _decode(append, B=batch, Hq=hq, Hkv=hkv, max_pages=max_pages, page=page, bt_sb=max_pages, ws=None, ws_bytes=0)
    assert rc == -28 and "workspace" in _err() or rc == -5, (rc, _err())
    return "chunks" if rc == -28 else "whole"


CHUNKED = [
    # test_gpu_decode_fp4: test_long_rows_of_small_batches, test_wide_table, test_each_form_of_launch
    (1, 16, 8, 157), (2, 16, 8, 313), (5, 16, 8, 188), (4, 16, 8, 4096), (65, 2, 1, 4096), (9, 32, 2, 260),
    # test_gpu_decode_fp4_forms: test_rows_that_outlast_a_window, test_queries_of_a_wide_range, test_chunks_captured_on_two_streams
    (200, 16, 8, 400), (1, 64, 64, 4300), (1, 384, 64, 4300), (1, 4, 2, 438), (1, 10, 2, 313), (1, 16, 8, 163), (1, 56, 8, 163), (3, 16, 8, 194), (3, 56, 8, 194),
    # test_gpu_fp4_limits: test_pool_without_pages_at_the_c_entry, test_graphs_that_share_their_memory_write_again
    (3, 16, 8, 4096), (3, 56, 8, 4096), (3, 128, 8, 4096), (2, 16, 8, 188), (2, 56, 8, 188),
]
EIGHT_WAVES = [
    # test_gpu_decode_fp4: test_ragged_rows, test_table_beyond_rows_capacity_is_clamped, test_captured_and_replayed
    (19, 16, 8, 44), (19, 9, 3, 44), (19, 32, 4, 44), (2, 16, 8, 4), (1, 16, 8, 57),
    # test_gpu_decode_fp4_forms: test_queries_of_a_wide_range, test_every_place_of_the_new_row (130 rows of 2 heads: four waves)
    (2, 4, 2, 19), (2, 14, 2, 9),
    # the first length that is cut is past 2048 tokens
    (1, 16, 8, 128), (32, 16, 8, 128), (1, 64, 8, 128),
    # test_gpu_fp4_limits: test_pool_without_pages_at_the_c_entry
    (3, 16, 8, 6), (3, 56, 8, 6),
]
FOUR_WAVES = [
    # test_gpu_decode_fp4: test_many_rows, test_each_form_of_launch, test_captured_and_replayed
    (300, 16, 8, 32), (300, 2, 2, 94), (64, 16, 8, 57), (80, 16, 8, 40),
    # test_gpu_decode_fp4_forms: test_every_place_of_the_new_row
    (130, 4, 2, 10),
    # test_gpu_fp4_limits: test_whole_rows_that_outlast_a_window, test_whole_rows_of_5_to_8_heads_in_four_waves,
    # test_pool_without_pages_at_the_c_entry
    (200, 16, 8, 290), (200, 48, 8, 290), (80, 32, 4, 60), (80, 20, 4, 60), (300, 7, 1, 60), (50, 48, 8, 60), (70, 28, 4, 6), (70, 8, 4, 6),
]


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("shape", CHUNKED)
def test_chunked(shape, append):
    assert _form(*shape, 16, append) == "chunks"


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up, and whole rows would be launched")
@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("shape", EIGHT_WAVES + FOUR_WAVES)
def test_whole_rows(shape, append):
    assert _form(*shape, 16, append) == "whole"


def test_the_lists_of_whole_rows_are_of_their_waves():
    assert all(b * hkv <= CUS and hq // hkv <= 8 for b, hq, hkv, _ in EIGHT_WAVES)
    assert all(b * hkv > CUS and hq // hkv <= 8 for b, hq, hkv, _ in FOUR_WAVES)
    for shapes in (CHUNKED, EIGHT_WAVES, FOUR_WAVES):          # both numbers of query heads that a wave may have
        assert {hq // hkv > 4 for _, hq, hkv, _ in shapes} == {False, True}


def test_the_workspace_query_names_one_for_whole_rows_too():
    """Shapes that are cut over the other pools and not over this one."""
    for shape in ((1, 16, 8, 57), (24, 16, 8, 96), (32, 16, 8, 128)):
        batch, hq, hkv, pages = shape
        assert _lib.lib().q3a_paged_decode_tree_workspace_bytes(batch, 1, hq, hkv, 128, pages, 16) > 0
