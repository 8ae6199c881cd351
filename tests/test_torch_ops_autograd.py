"""What autograd sees of the 8-bit pool's and the tree attention's ops: a backward is refused, not left out, and what writes into
caches counts as in-place.  On meta tensors, whose outputs have shapes only; the GPU part runs the ops."""
import pytest
import torch

import q3attn


def _args(device, B=2, N=3, Hq=4, Hkv=2):
    f = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device=device)
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)
    pool = q3attn.fp8_cache(4, 16, Hkv, device=device)
    return dict(q=f(B, Hq, 128), k=f(B, Hkv, 128), v=f(B, Hkv, 128), qn=f(B, N, Hq, 128), kn=f(B, N, Hkv, 128), vn=f(B, N, Hkv, 128),
                pool=pool, bf16=(f(4, 16, Hkv, 128), f(4, 16, Hkv, 128)), lens=i(B), table=i(B, 4),
                slots=torch.zeros((B,), dtype=torch.int64, device=device))


def _decode(a):
    return q3attn.paged_decode_fp8(a["q"], *a["pool"], a["lens"], a["table"], 0.1)


def _append(a):
    return q3attn.paged_decode_fp8_append(a["q"], a["k"], a["v"], *a["pool"], a["lens"], a["table"], 0.1)


def _tree(a):
    return q3attn.paged_decode_tree(a["qn"], a["kn"], a["vn"], None, *a["bf16"], a["lens"], a["table"], 0.1)


def _tree_fp8(a):
    return q3attn.paged_decode_tree(a["qn"], a["kn"], a["vn"], None, *a["pool"][:2], a["lens"], a["table"], 0.1, *a["pool"][2:])


DEVICES = ["meta", pytest.param("cuda", marks=pytest.mark.gpu)]
NEED = [(_decode, "q"), (_append, "q"), (_append, "k"), (_append, "v"), (_tree, "qn"), (_tree, "vn"), (_tree_fp8, "qn"), (_tree_fp8, "kn")]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("call,name", NEED)
def test_a_backward_is_refused(call, name, device):
    a = _args(device)
    a[name] = a[name].float().requires_grad_().to(torch.bfloat16)     # not a leaf, as a projection's output
    out = call(a)
    assert out.requires_grad
    with pytest.raises(RuntimeError, match="paged_decode.* is not implemented"):
        out.sum().backward()
    with torch.no_grad():
        assert not call(a).requires_grad
    assert not call(_args(device)).requires_grad


@pytest.mark.parametrize("device", DEVICES)
def test_writes_count_as_in_place(device):
    a = _args(device)
    versions = lambda: [t._version for t in a["pool"]]
    v0 = versions()
    q3attn.paged_write_fp8(a["k"], a["v"], a["slots"], *a["pool"])
    v1 = versions()
    assert all(x > y for x, y in zip(v1, v0))
    _append(a)
    v2 = versions()
    assert all(x > y for x, y in zip(v2, v1))
    with torch.no_grad():
        q3attn.paged_write_fp8(a["k"], a["v"], a["slots"], *a["pool"])
    with torch.inference_mode():
        q3attn.paged_write_fp8(a["k"], a["v"], a["slots"], *a["pool"])
    v3 = versions()
    assert all(x > y + 1 for x, y in zip(v3, v2))
    inputs = [a[n] for n in ("q", "k", "v", "qn", "kn", "vn", "lens", "table", "slots")] + list(a["bf16"])
    before = [t._version for t in inputs]
    q3attn.paged_read_fp8(*a["pool"], a["slots"])
    for call in (_decode, _tree, _tree_fp8):
        call(a)
    assert versions() == v3 and [t._version for t in inputs] == before


@pytest.mark.parametrize("device", DEVICES)
def test_inference_tensors(device):
    with torch.inference_mode():
        a = _args(device)
        q3attn.paged_write_fp8(a["k"], a["v"], a["slots"], *a["pool"])
        k, v = q3attn.paged_read_fp8(*a["pool"], a["slots"])
        outs = [k, v] + [call(a) for call in (_decode, _append, _tree, _tree_fp8)]
    assert all(t.is_inference() and not t.requires_grad for t in outs)


def test_fakes_have_the_ops_shapes():
    a = _args("meta")
    assert _decode(a).shape == _append(a).shape == a["q"].shape and _tree(a).shape == _tree_fp8(a).shape == a["qn"].shape
    a["qn"] = torch.zeros((2, 4, 3, 128), dtype=torch.bfloat16, device="meta").transpose(1, 2)
    a["q"] = torch.zeros((4, 2, 128), dtype=torch.bfloat16, device="meta").transpose(0, 1)
    for out in (_decode(a), _append(a), _tree(a), _tree_fp8(a)):
        assert out.is_contiguous() and out.dtype == torch.bfloat16
    k, v = q3attn.paged_read_fp8(*a["pool"], a["slots"])
    assert k.shape == v.shape == (2, 2, 128) and k.is_contiguous() and v.is_contiguous() and k.dtype == v.dtype == torch.bfloat16
