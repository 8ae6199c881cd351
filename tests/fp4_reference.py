"""Plain 64-bit restatement of the 4-bit K/V pool's row format, on the CPU, for the tests.  (Attention over a paged pool's values and
tables of random pages are fp8_reference's.)"""
import math

import numpy as np
import torch

D = 128
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantise(x):
    """Rows [..., 128] -> (values of the codes before the scale, float64 [..., 128], exponent bytes int64 [..., 4]), from the
    definition.  Blocks with an element that is not finite have byte 255 and codes 0."""
    x = x.double().unflatten(-1, (4, 32))
    fine = torch.isfinite(x).all(-1)
    top = torch.where(fine[..., None], x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.full(top.shape, -125, dtype=torch.int64)
    for n in range(-125, 125):                                # the least n with top <= 7 * 2^n, at most 125
        e = torch.where(top > 7.0 * 2.0 ** n, n + 1, e)
    y = (x / torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None]).numpy()
    dist = np.abs(np.abs(np.where(np.isfinite(y), y, 0))[..., None] - GRID)      # nearest code, ties to the even one
    code = np.where(dist == dist.min(-1, keepdims=True), np.arange(8) % 2, 2).argmin(-1)
    v = torch.from_numpy(np.copysign(GRID[code], np.where(np.isnan(y), 1.0, y)))
    v = torch.where(fine[..., None], v, torch.zeros_like(v))
    return v.flatten(-2), torch.where(fine, e + 127, 255)


def pack(v):
    """Code values [..., 128] -> bytes [..., 64]."""
    a = np.abs(v.numpy())
    code = torch.from_numpy(np.searchsorted(GRID, a)).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4)


def values(codes, exps):
    """Bytes [..., 64] and exponent bytes [..., 4] -> float64 [..., 128]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    grid = torch.from_numpy(np.concatenate([GRID, -GRID]))
    e = exps.long()
    f = torch.where(e == 255, math.nan, torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double() - 127.0))
    return grid[c] * f.repeat_interleave(32, -1)


def pool_values(cache, scale):
    """[pages, page, Hkv, 128] float64 values of a pool."""
    return values(cache.cpu(), scale.cpu().permute(0, 3, 1, 2))


def fill_pool(pages, page, hkv, head_major, seed, device):
    """(k_cache, v_cache, k_scale, v_scale): a pool of random rows on ``device``."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for spread in (0.3, 1.0):
        x = torch.randn((pages, page, hkv, D), generator=g) * torch.exp(spread * torch.randn((pages, page, hkv, 1), generator=g))
        v, e = quantise(x.to(torch.bfloat16))
        code = pack(v).to(device)
        if head_major:
            code = code.transpose(1, 2).contiguous().transpose(1, 2)
        out.append((code, e.to(torch.uint8).permute(0, 2, 3, 1).contiguous().to(device)))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def assert_close(got, want, spread, score_err=5e-4):
    """Elementwise: half a bf16 step (2^-8) of the result for its rounding; of spread = sum p |v| / sum p, 2^-14 for the probabilities
    (two bf16 numbers each, 2^-15 left, in the sum too), 3e-4 for fp32 sums of up to 5000 terms (5000 * 2^-24), and score_err for the
    fp32 scores (128 products of at most ~60 in all: 128 * 2^-24 * 60 < 5e-4) and exp2."""
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -14 + 3e-4 + score_err) * spread * (1 + 2.0 ** -7) + 1e-30
    bad = ((got - want).abs() > tol) & fine
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol)[fine].max()), bad.nonzero()[:5].tolist())
