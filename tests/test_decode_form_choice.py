"""CPU tests of the form of launch that decode over the 8-bit pool and tree attention choose from a call's shape: whole rows need no
workspace, chunks of rows do.  The shapes are those of the GPU tests that are meant for one form, so that a rule that moves does not
leave a form untested."""
import pytest
import torch

import q3attn
from q3attn import _lib


def _workspace(batch, nodes, hq, hkv, max_pages, page=16):
    return _lib.lib().q3a_paged_decode_tree_workspace_bytes(batch, nodes, hq, hkv, 128, max_pages, page)


def _pages(tokens):
    return -(-tokens // 16)


CHUNKED = [
    # test_gpu_decode_forms: test_chunks_of_many_rows, test_append_to_many_rows, test_chunks_of_trees, test_scales_that_are_not_positive,
    # test_graphs_that_share_their_memory, test_trees_on_two_streams
    (65, 1, 2, 1, 4096), (130, 1, 4, 2, 2048), (1024, 1, 2, 1, 512), (63, 1, 16, 8, 600), (130, 1, 2, 1, 2048),
    (3, 40, 4, 2, _pages(2000)), (1, 130, 1, 1, _pages(3000)), (4, 17, 6, 3, _pages(1500)), (3, 3, 16, 1, _pages(2500)),
    (1, 1, 4, 2, _pages(1501)), (1, 5, 4, 2, _pages(1500)), (2, 1, 16, 8, _pages(2001)), (1, 20, 4, 2, _pages(2000)),
    (3, 20, 4, 2, _pages(1500)),
    # test_gpu_decode_fp8: test_long_rows_of_small_batches, test_wide_table, test_captured_and_replayed, test_two_streams
    (1, 1, 16, 8, _pages(2501)), (2, 1, 16, 8, _pages(5001)), (5, 1, 16, 8, _pages(3001)), (4, 1, 16, 8, 4096), (1, 1, 16, 8, _pages(901)),
    # test_gpu_decode_tree: test_long_contexts, test_captured_and_replayed
    (2, 6, 4, 2, _pages(3000)), (3, 5, 4, 2, _pages(900)),
]
WHOLE = [
    # test_gpu_decode_forms: test_rows_in_the_order_of_their_lengths, test_append_to_many_rows, test_trees_of_many_rows,
    # test_graphs_that_share_their_memory, test_a_row_gets_the_same_bits_whatever_the_batch_holds,
    # test_long_rows_whose_query_rows_fill_the_chip
    (5, 1, 64, 64, _pages(900)), (64, 1, 8, 8, _pages(900)), (256, 1, 2, 2, _pages(1000)), (300, 1, 2, 2, _pages(1500)),
    (520, 1, 1, 1, _pages(1400)), (300, 1, 4, 2, 80), (270, 3, 4, 2, 48), (300, 1, 16, 8, _pages(599)), (120, 1, 8, 4, 32),
    (1, 64, 256, 16, 4096),
    # test_gpu_decode_fp8: test_ragged_rows, test_many_rows, test_captured_and_replayed
    (19, 1, 16, 8, _pages(701)), (300, 1, 16, 8, _pages(500)), (80, 1, 16, 8, _pages(633)),
    # test_gpu_decode_tree: test_trees, test_chain
    (6, 3, 16, 8, _pages(100)), (6, 17, 4, 2, _pages(100)), (4, 20, 4, 2, _pages(150)),
]


@pytest.mark.parametrize("shape", CHUNKED)
def test_chunked(shape):
    assert _workspace(*shape) > 0


@pytest.mark.parametrize("shape", WHOLE)
def test_whole_rows(shape):
    assert _workspace(*shape) == 0


def test_cpu_tensors_are_refused_by_the_ops_themselves():
    pool = q3attn.fp8_cache(2, device="cpu")
    x = torch.zeros((1, 8, 128), dtype=torch.bfloat16)
    q = torch.zeros((1, 16, 128), dtype=torch.bfloat16)
    n, bt = torch.zeros((1,), dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32)
    slot = torch.zeros((1,), dtype=torch.int64)
    for call in (lambda: q3attn.paged_write_fp8(x, x, slot, *pool), lambda: q3attn.paged_read_fp8(*pool, slot),
                 lambda: q3attn.paged_decode_fp8(q, *pool, n, bt, 1.0),
                 lambda: q3attn.paged_decode_fp8_append(q, x, x, *pool, n, bt, 1.0),
                 lambda: q3attn.paged_decode_tree(q[:, None], x[:, None], x[:, None], None, *pool[:2], n, bt, 1.0, *pool[2:])):
        with pytest.raises(RuntimeError, match="must be on a GPU"):
            call()
