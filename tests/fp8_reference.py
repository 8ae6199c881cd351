"""Plain 64-bit restatements of the 8-bit K/V pool's row format and of attention over a paged pool, on the CPU, for the tests."""
import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn
D = 128


def quantise(x):
    """Rows [..., 128] -> (code values float64, exponent bytes int64), from the definition."""
    x = x.double()
    top = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.full(top.shape, -117, dtype=torch.int64)
    for n in range(-117, 121):                                # the least n with top <= 448 * 2^n
        e = torch.where(top > 448.0 * 2.0 ** n, n + 1, e)
    y = x / torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None]
    spacing = torch.pow(torch.tensor(2.0, dtype=torch.float64),
                        torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    code = torch.round(y / spacing) * spacing                 # torch.round: to even
    code = torch.where((e == 120)[..., None], code.clamp(-240, 240), code)   # 256 * 2^120 is over the largest bf16
    code = torch.where(torch.isfinite(x), code, torch.full_like(code, math.nan))
    return code, e + 127


def pool_values(cache, scale):
    """[pages, page, Hkv, D] float64 values of a pool on the CPU; bf16 pools as they are."""
    if scale is None:
        return cache.cpu().double()
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), scale.cpu().double() - 127.0)
    return cache.cpu().contiguous().view(torch.uint8).view(E4M3).float().double() * s.transpose(1, 2)[..., None]


def fill_pool(pages, page, hkv, fp8, head_major, seed, device):
    """(k_cache, v_cache, k_scale, v_scale): a pool of random rows on ``device`` (scales None for bf16)."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for spread in (0.3, 1.0):
        x = torch.randn((pages, page, hkv, D), generator=g) * torch.exp(spread * torch.randn((pages, page, hkv, 1), generator=g))
        x = x.to(torch.bfloat16)
        scale = None
        if fp8:
            code, s = quantise(x)
            x, scale = code.float().to(E4M3).view(torch.uint8), s.to(torch.uint8).transpose(1, 2).contiguous().to(device)
        x = x.to(device)
        if head_major:
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        out.append((x.view(E4M3) if fp8 else x, scale))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def table_for(lens, page, pages, width, seed):
    """A random table [B, width] whose rows hold ceil(len / page) distinct pages each, -1 behind."""
    rng = np.random.default_rng(seed)
    ids, at = rng.permutation(pages), 0
    t = np.full((len(lens), width), -1, np.int32)
    for b, n in enumerate(lens):
        used = -(-max(int(n), 0) // page)
        t[b, :used] = ids[at:at + used]
        at += used
    return torch.from_numpy(t)


def attention(q, kvals, vvals, lens, table, scale, own=None):
    """(out, spread) [B, N, Hq, D] float64: attention over each row's cached tokens and ``own`` = (k, v, mask [B, N, N]);
    spread = sum p |v| / sum p, which bounds what rounding the probabilities can change.  Rows with lens < 0 are zeros."""
    q = q.cpu().double()
    B, N, Hq, _ = q.shape
    P, page, Hkv, _ = kvals.shape
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        n = int(lens[b])
        if n < 0:
            continue
        tok = torch.arange(min(n, table.shape[1] * page))
        ids = table[b].long()[tok // page] if len(tok) else tok
        live = (ids >= 0) & (ids < P)
        ids, off = ids[live], (tok % page)[live]
        k, v = kvals[ids, off], vvals[ids, off]                               # [n, Hkv, D]
        see = torch.ones((N, k.shape[0]), dtype=torch.bool)
        if own is not None:
            k, v = torch.cat([k, own[0][b].cpu().double()]), torch.cat([v, own[1][b].cpu().double()])
            see = torch.cat([see, own[2][b].cpu()], 1)
        for h in range(Hq):
            kk, vv = k[:, h // (Hq // Hkv)], v[:, h // (Hq // Hkv)]
            for i in range(N):
                w = see[i]
                if not w.any():
                    continue
                p = torch.softmax(kk[w] @ q[b, i, h] * scale, 0)
                out[b, i, h] = p @ vv[w]
                spread[b, i, h] = p @ vv[w].abs()
    return out, spread


def assert_close(got, want, spread, score_err=5e-4):
    """Elementwise: half a bf16 step (2^-8) of the result for its rounding, and of the spread for that of the probabilities;
    score_err of the spread for the fp32 scores (128 products of at most ~60 in all: 128 * 2^-24 * 60 < 5e-4) and exp2."""
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + score_err) * spread * (1 + 2.0 ** -7) + 1e-30
    bad = ((got - want).abs() > tol) & fine
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol)[fine].max()), bad.nonzero()[:5].tolist())
