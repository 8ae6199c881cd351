"""How many launches a copy of pages takes: one for up to 128 caches of up to four shapes, in whatever order the list has them."""
import ctypes

import numpy as np
import pytest
import torch

import q3attn
from q3attn import _lib
from test_gpu_paged_moves import _bytes, _check_copy, _random, _want_copy

pytestmark = pytest.mark.gpu


def _launches(caches, dev):
    """Nodes of a captured copy, which is replayed and compared."""
    src, dst = ([3, 0, 5], [1, 2, 4])
    ids = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (src, dst)]
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        q3attn.paged_copy(caches, *ids)
    count = ctypes.c_size_t(0)
    assert _lib.lib().hipGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(count)) == 0
    graph.instantiate()
    for seed in range(2):
        for i, c in enumerate(caches):
            c.view(torch.uint8).copy_(_random(c.view(torch.uint8).shape, 100 * seed + i, dev))
        want = _want_copy(caches, src, dst)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(_bytes(c), w) for c, w in zip(caches, want))
    return count.value


def _layers(kinds, layers, dev):
    """The layers' caches one layer after the other: K, V and their scales."""
    make = {"bf16": lambda: [torch.zeros((7, 16, 2, 128), dtype=torch.bfloat16, device=dev) for _ in range(2)],
            "fp8": lambda: q3attn.fp8_cache(7, 16, 2, device=dev), "fp4": lambda: q3attn.fp4_cache(7, 16, 2, device=dev)}
    return [t for _ in range(layers) for kind in kinds for t in make[kind]()]


@pytest.mark.parametrize("kinds,layers,launches", [(["fp8"], 28, 1), (["fp4"], 28, 1), (["bf16"], 28, 1), (["fp8", "fp4"], 16, 1),
                                                   (["fp4"], 40, 2), (["bf16"], 150, 3)])
def test_layers_in_order(cuda_device, kinds, layers, launches):
    caches = _layers(kinds, layers, cuda_device)
    count = _launches(caches, cuda_device)
    assert count == launches == -(-len(caches) // 128)


def test_shuffled_shapes(cuda_device):
    """Any order of shapes, and more of them than a launch takes."""
    shapes = [(7, 16, 2, 64), (9, 16, 4, 64), (6, 48), (8, 16)]
    order = np.random.default_rng(0).permutation(40).tolist()
    count = _launches([_random(shapes[i % 4], i, cuda_device) for i in order], cuda_device)
    assert count == 1
    many = [_random((6 + i % 5, 16 * (1 + i % 6)), i, cuda_device) for i in np.random.default_rng(1).permutation(60).tolist()]
    _check_copy(many, [0, 4, 5, 9], [2, 3, 1, 7])
    views = [t for i in range(3) for both in [_random((9, 2, 16, 4, 64), i, cuda_device)]
             for t in (both[:, 0], _random((7, 16), 50 + i, cuda_device), both[:, 1, :, 1:3])]
    _check_copy([v for i, v in enumerate(views) if i % 3 != 2], [0, 5], [2, 3])
    _check_copy([v for i, v in enumerate(views) if i % 3 != 0], [1, 6], [0, 4])
