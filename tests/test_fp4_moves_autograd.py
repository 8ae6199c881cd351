"""What autograd sees of the 4-bit pool's ops and of the moves of pages and tokens: a backward is refused, not left out, also one through a
cache that was moved in, and what writes into caches counts as in-place.  On meta tensors, whose outputs have shapes only; the GPU part runs
the ops."""
import pytest
import torch

import q3attn

DEVICES = ["meta", pytest.param("cuda", marks=pytest.mark.gpu)]


def _args(device, B=2, Hq=4, Hkv=2):
    f = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device=device)
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)
    return dict(q=f(B, Hq, 128), k=f(B, Hkv, 128), v=f(B, Hkv, 128), pool=q3attn.fp4_cache(4, 16, Hkv, device=device),
                fp8=q3attn.fp8_cache(4, 16, Hkv, device=device), bf16=[f(4, 16, Hkv, 128) for _ in range(3)], lens=i(B), table=i(B, 4),
                slots=torch.zeros((B,), dtype=torch.int64, device=device), src=i(1), dst=i(1) + 1,
                keep=torch.ones((B, 8), dtype=torch.bool, device=device))


def _decode(a):
    return q3attn.paged_decode_fp4(a["q"], *a["pool"], a["lens"], a["table"], 0.1)


def _append(a):
    return q3attn.paged_decode_fp4_append(a["q"], a["k"], a["v"], *a["pool"], a["lens"], a["table"], 0.1)


def _copy(a, caches):
    q3attn.paged_copy(caches, a["src"], a["dst"])


def _compact(a, caches):
    q3attn.paged_compact(caches, a["keep"], a["lens"], a["table"])


MOVES = [_copy, _compact]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("call,name", [(_decode, "q"), (_append, "q"), (_append, "k"), (_append, "v")])
def test_a_backward_is_refused(call, name, device):
    a = _args(device)
    a[name] = a[name].float().requires_grad_().to(torch.bfloat16)     # not a leaf, as a projection's output
    out = call(a)
    assert out.requires_grad
    with pytest.raises(RuntimeError, match="paged_decode_fp4.* is not implemented"):
        out.sum().backward()
    with torch.no_grad():
        assert not call(a).requires_grad
    assert not call(_args(device)).requires_grad


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("move", MOVES)
@pytest.mark.parametrize("which", [0, 2])
def test_a_backward_through_a_moved_cache_is_refused(move, which, device):
    """The pages that were written over no longer are what the cache's history says."""
    a = _args(device)
    leaf = a["bf16"][which].clone().requires_grad_()
    a["bf16"][which] = cache = leaf * 2
    move(a, a["bf16"])
    assert [t.requires_grad for t in a["bf16"]] == [i == which for i in range(3)]
    with pytest.raises(RuntimeError, match="paged_co.* is not implemented"):
        cache.float().sum().backward()
    assert leaf.grad is None


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("move", MOVES)
def test_a_backward_through_a_moved_view_is_refused(move, device):
    """A layer of a stack: the stack's history ends there as well."""
    a = _args(device)
    leaf = torch.zeros((2, 4, 16, 2, 128), dtype=torch.bfloat16, device=device, requires_grad=True)
    stack = leaf * 2
    move(a, [stack[1]])
    with pytest.raises(RuntimeError, match="paged_co.* is not implemented"):
        stack.float().sum().backward()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("move", MOVES)
def test_leaves_that_require_gradients_are_refused(move, device):
    a = _args(device)
    a["bf16"][1].requires_grad_()
    before = [t._version for t in a["bf16"]]
    with pytest.raises(RuntimeError, match="leaf"):
        move(a, a["bf16"])
    assert [t._version for t in a["bf16"]] == before
    with torch.no_grad():                                             # as torch's own in-place operations
        move(a, a["bf16"])
    assert a["bf16"][1].requires_grad and a["bf16"][1].is_leaf


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("move", MOVES)
def test_a_cache_saved_for_a_backward_is_noticed(move, device):
    a = _args(device)
    w = torch.ones((), dtype=torch.bfloat16, device=device, requires_grad=True)
    y = a["bf16"][0] * w
    move(a, a["bf16"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


@pytest.mark.parametrize("device", DEVICES)
def test_writes_count_as_in_place(device):
    a = _args(device)
    versions = lambda ts: [t._version for t in ts]
    every = [*a["pool"], *a["fp8"], *a["bf16"]]
    calls = [(lambda: q3attn.paged_write_fp4(a["k"], a["v"], a["slots"], *a["pool"]), a["pool"]), (lambda: _append(a), a["pool"]),
             (lambda: _copy(a, every), every), (lambda: _copy(a, a["bf16"][1:]), a["bf16"][1:]), (lambda: _compact(a, a["bf16"]), a["bf16"]),
             (lambda: q3attn.paged_compact(a["pool"][:2], a["keep"], a["lens"], a["table"], a["pool"][2:]), a["pool"]),
             (lambda: q3attn.paged_compact(a["fp8"][:1], a["keep"], a["lens"], a["table"], a["fp8"][2:3]), (a["fp8"][0], a["fp8"][2]))]
    inputs = [a[n] for n in ("q", "k", "v", "lens", "table", "slots", "src", "dst", "keep")]
    start = versions(inputs)
    for mode in (torch.enable_grad, torch.no_grad, torch.inference_mode):
        for call, written in calls:
            others = [t for t in every if not any(t is w for w in written)]
            before, rest = versions(written), versions(others)
            with mode():
                call()
            assert all(x > y for x, y in zip(versions(written), before)) and versions(others) == rest
    before = versions(every)
    q3attn.paged_read_fp4(*a["pool"], a["slots"])
    _decode(a)
    assert versions(every) == before and versions(inputs) == start


@pytest.mark.parametrize("device", DEVICES)
def test_inference_tensors(device):
    with torch.inference_mode():
        a = _args(device)
        q3attn.paged_write_fp4(a["k"], a["v"], a["slots"], *a["pool"])
        outs = [*q3attn.paged_read_fp4(*a["pool"], a["slots"]), _decode(a), _append(a)]
        _copy(a, [*a["pool"], *a["bf16"]])
        outs.append(q3attn.paged_compact(a["bf16"], a["keep"], a["lens"], a["table"]))
    assert all(t.is_inference() and not t.requires_grad for t in outs)


def test_fakes_have_the_ops_shapes():
    a = _args("meta")
    assert _decode(a).shape == _append(a).shape == a["q"].shape
    k, v = q3attn.paged_read_fp4(*a["pool"], a["slots"])
    assert k.shape == v.shape == (2, 2, 128) and k.is_contiguous() and v.is_contiguous() and k.dtype == v.dtype == torch.bfloat16
    n = q3attn.paged_compact(a["bf16"], a["keep"], a["lens"], a["table"])
    assert n.shape == (2,) and n.dtype == torch.int32
