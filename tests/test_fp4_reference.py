"""The 4-bit pool's restatement for the tests against the format's own properties (CPU)."""
import numpy as np
import torch

from fp4_reference import GRID, pack, quantise, values


def test_codes_stand_for_themselves_at_any_scale():
    for e in (-125, -3, 0, 125):
        x = torch.from_numpy(np.resize(np.concatenate([GRID, -GRID]), 128)) * 2.0 ** e
        v, s = quantise(x[None])
        assert (s == e + 127).all()
        assert torch.equal(values(pack(v), s.to(torch.uint8))[0], x)


def test_ties_and_borders():
    x = torch.zeros(128, dtype=torch.float64)
    x[:10] = torch.tensor([7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0], dtype=torch.float64)
    v, s = quantise(x[None])
    assert s[0, 0] == 127 and s[0, 1] == 2
    assert v[0, :10].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -4]
    x[0] = 7.0625                                             # the next bf16: the next scale
    assert quantise(x[None])[1][0, 0] == 128


def test_error_is_at_most_half_a_step():
    x = torch.randn((2000, 128), generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    v, s = quantise(x)
    got = values(pack(v), s.to(torch.uint8))
    top = x.double().abs().unflatten(-1, (4, 32)).amax(-1).repeat_interleave(32, -1)
    assert ((got - x.double()).abs() <= top / 3.5).all()      # half of the widest step, 1, at a scale of at least top / 7 ... top / 3.5
    assert ((got - x.double()).pow(2).mean() / x.double().pow(2).mean()) < 0.014


def test_blocks_that_are_not_finite():
    x = torch.ones((1, 128))
    x[0, 40] = float("inf")
    x[0, 127] = float("nan")
    v, s = quantise(x)
    assert s[0].tolist()[1::2] == [255, 255] and (v[0, 32:64] == 0).all()
    got = values(pack(v), s.to(torch.uint8))
    assert torch.isnan(got[0, 32:64]).all() and torch.isnan(got[0, 96:]).all() and (got[0, :32] == 1).all()
