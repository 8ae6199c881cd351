"""The 4-bit K/V cache and the moves of cached tokens, as timed cases.

A row of the 4-bit pool (one token of one KV head, 128 values) is held as e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives), two a byte, and one exponent byte s for each 32 of them: value = code * 2^(s-127), with 2^(s-127) the smallest power
of two that takes the 32 values' largest magnitude to at most 7 (6 is the largest code, and the nearest to all up to 7).

  store    k and v of T new tokens into the pool, token t at slot page * page_size + offset (negative: not written), and back as
           the bf16 rows that the pool now stands for, which is what a prefill attends
  read     T slots of the pool back to bf16
  decode   one query token a row over the row's cached tokens; with ``append`` the step's k and v are written first, and what the
           pool holds of them is read back
  copy     whole pages to other pages, in every layer's K and V at once: forks of a prompt, pages moved together
  compact  the kept tokens of each row to the front of its pages, in order, in every layer's K and V at once

With ``own`` the q3attn operators run, else the same in elementary torch operations.
"""
from __future__ import annotations

import math
import os
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False

D = 128
BLOCK = 32
SCALE = D ** -0.5
DEV = "cuda"
BF = torch.bfloat16
E4 = torch.float8_e4m3fn
E_MIN, E_MAX = -125, 125   # the smallest code is still a normal number, and the largest still a finite bf16


def listed():
    return [
        # One decode step's K and V of a full server: 576 seats, a tenth of them empty.
        {"name": "store_step_576", "kind": "store", "tokens": 576, "pads": 58, "page": 16, "hkv": 8, "head_major": True},
        # A burst of 64 long prompts.
        {"name": "store_prompts_64x1700", "kind": "store", "tokens": 108800, "pads": 0, "page": 16, "hkv": 8,
         "head_major": True},
        # A cached voice prefix of 77 tokens read back for a prefill, token-major pool of 256-token pages.
        {"name": "read_prefix_77", "kind": "read", "tokens": 77, "pads": 0, "page": 256, "hkv": 8, "head_major": False},
        # 32 seats moved out of the pool.
        {"name": "read_seats_32x1100", "kind": "read", "tokens": 35200, "pads": 11, "page": 16, "hkv": 8,
         "head_major": True},
        # One stream speaking: where launches and latency are the time.
        {"name": "decode_1row", "kind": "decode", "append": False, "rows": 1, "pads": 0, "lo": 700, "hi": 1100, "page": 16,
         "hq": 16, "hkv": 8, "head_major": True, "seed_ctx": 1},
        # A lightly loaded server with the step's write, on a token-major pool.
        {"name": "decode_24rows_append", "kind": "decode", "append": True, "rows": 24, "pads": 2, "lo": 100, "hi": 1500,
         "page": 16, "hq": 16, "hkv": 8, "head_major": False, "seed_ctx": 2},
        # The full server: 576 seats, a tenth of them empty, log-uniform contexts.
        {"name": "decode_576rows_append", "kind": "decode", "append": True, "rows": 576, "pads": 58, "lo": 64, "hi": 1800,
         "page": 16, "hq": 16, "hkv": 8, "head_major": True, "seed_ctx": 5},
        # Few rows of very long contexts, 8 query heads to a KV head.
        {"name": "decode_5rows_long", "kind": "decode", "append": False, "rows": 5, "pads": 0, "lo": 20000, "hi": 65000,
         "page": 64, "hq": 32, "hkv": 4, "head_major": True, "seed_ctx": 6},
        # Three samples forked off one prompt: its last, partly filled page, in 28 layers of the bf16 pool.
        {"name": "copy_fork_3", "kind": "copy", "fork": True, "fp8": False, "layers": 28, "pairs": 3, "page": 16, "hkv": 8},
        # The pool's pages moved together after a busy hour: 600 pages in 28 layers of the 8-bit pool.
        {"name": "copy_pages_600", "kind": "copy", "fork": False, "fp8": True, "layers": 28, "pairs": 600, "page": 16, "hkv": 8},
        # One long stream that goes on with its first tokens and its latest.
        {"name": "compact_1row_window", "kind": "compact", "window": True, "fp8": False, "layers": 28, "rows": 1, "lo": 700,
         "hi": 1100, "page": 16, "hkv": 8, "seed_ctx": 11},
        # 48 seats that let go of the tokens that were hardly attended.
        {"name": "compact_48rows_evict", "kind": "compact", "window": False, "fp8": True, "layers": 28, "rows": 48, "lo": 300,
         "hi": 1800, "page": 16, "hkv": 8, "seed_ctx": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "read", "decode", "decode", "copy", "compact"])
    page, hkv = rng.choice([16, 16, 32, 64, 256]), rng.choice([8, 8, 8, 4, 2])
    case = {"kind": kind, "page": page, "hkv": hkv}
    if kind in ("store", "read"):
        tokens = _log_int(rng, 1, 100000 if kind == "store" else 33000)
        return {**case, "tokens": tokens, "pads": rng.randrange(0, tokens // 8 + 1), "head_major": rng.random() < 0.6}
    if kind == "decode":
        hi = _log_int(rng, 16, 30000)
        lo = max(1, int(hi * rng.uniform(0.05, 1.0)))
        rows = max(1, min(_log_int(rng, 1, 576), int(240000 / (0.5 * (lo + hi)))))
        return {**case, "append": rng.random() < 0.5, "rows": rows, "pads": rng.randrange(0, rows // 8 + 1), "lo": lo, "hi": hi,
                "hq": hkv * rng.choice([1, 2, 2, 4, 8]), "head_major": rng.random() < 0.6, "seed_ctx": rng.randrange(1 << 20)}
    fp8, layers = rng.random() < 0.5, rng.choice([1, 5, 28, 28])
    case |= {"fp8": fp8, "layers": layers}
    if kind == "copy":
        return {**case, "fork": rng.random() < 0.4, "pairs": _log_int(rng, 1, 9600 * 8 // (page * hkv))}
    hi = _log_int(rng, 20, 4000)
    lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
    rows = max(1, min(_log_int(rng, 1, 256), (24000 if fp8 else 14000) // hi))
    return {**case, "window": rng.random() < 0.5, "rows": rows, "lo": lo, "hi": hi, "seed_ctx": rng.randrange(1 << 20)}


# ---------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _keys(shape, g):
    """Normalised keys: rows of unit RMS with a norm weight that differs from dim to dim."""
    x = torch.randn(shape, generator=g, device=DEV)
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)
    return (x * (0.5 + torch.rand(shape[-1], generator=g, device=DEV))).to(BF)


def _values(shape, g):
    """Values whose rows differ in size, as the projections of loud and quiet tokens do."""
    x = torch.randn(shape, generator=g, device=DEV)
    return (x * torch.exp(torch.randn(shape[:-1] + (1,), generator=g, device=DEV))).to(BF)


def _pow2(e):
    """2^e in fp32 for -126 <= e <= 127, from its bits (pow need not give a power of two exactly)."""
    return (e.int() + 127 << 23).view(torch.float32)


def _codes(x):
    """Rows of x [..., D] as (packed e2m1 codes [..., D / 2], exponent bytes [..., D / 32]); the inputs are finite."""
    x = x.float().unflatten(-1, (D // BLOCK, BLOCK))
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m == 0, E_MIN, torch.clamp(e - 3 + (m > 0.875).int(), E_MIN, E_MAX))
    y = x * _pow2(-e)[..., None]
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.clamp(torch.round(a / step) * step, max=6.0)
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, 0.5 * a + 4)).to(torch.uint8)
    code = (code | (torch.signbit(y).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _pool4(pages, case, g):
    """K and V pools filled with earlier tokens, [pages, page, hkv, D / 2] bytes, and the exponents [pages, hkv, D / 32, page]."""
    p, h = case["page"], case["hkv"]
    shape = (pages, h, p) if case["head_major"] else (pages, p, h)
    step = max(1, 65536 // p)
    pools, scales = [], []
    for make in (_keys, _values):
        pool = torch.empty(shape + (D // 2,), dtype=torch.uint8, device=DEV)
        scale = torch.empty((pages, h, D // BLOCK, p), dtype=torch.uint8, device=DEV)
        for c in range(0, pages, step):
            x, e = _codes(make((min(step, pages - c),) + shape[1:] + (D,), g))
            pool[c:c + step] = x
            scale[c:c + step] = e.transpose(2, 3) if case["head_major"] else e.permute(0, 2, 3, 1)
        pools.append(pool.transpose(1, 2) if case["head_major"] else pool)
        scales.append(scale)
    return pools + scales


def _contexts(case):
    """Tokens attended in each row, this step's included; the padded rows (0) are the last.  They belong to the case, not
    to the seed, so that every pass of a case does the same work."""
    rng = np.random.default_rng(case["seed_ctx"])
    lo, hi, pads = case["lo"], case["hi"], case.get("pads", 0)
    live = case["rows"] - pads
    c = np.rint(np.exp(rng.uniform(math.log(lo), math.log(hi), size=live))) if hi > 4 * lo else rng.integers(lo, hi + 1, live)
    return np.concatenate([c.astype(np.int64), np.zeros(pads, np.int64)])


def _kept(case):
    """Which tokens a compaction keeps, [rows, longest]; of the case as the contexts are."""
    ctx = _contexts(case)
    rng = np.random.default_rng(case["seed_ctx"] + 1)
    at, n = np.arange(int(ctx.max()))[None], ctx[:, None]
    if case["window"]:
        return (at < n) & ((at < 4) | (at >= n - np.maximum(1, n * 6 // 10)))    # the first 4 and the latest 60 %
    # the latest eighth, and of the others those whose weight is above a cut that differs from row to row
    return (at < n) & ((at >= n - n // 8) | (rng.random((len(ctx), at.shape[1])) < rng.uniform(0.3, 0.9, (len(ctx), 1))))


def _tables(ctx, page, rng):
    """The rows' tables over scattered pages (page 0 is no row's), and how many pages there are."""
    used = -(-ctx // page)
    width = (256 * -(-int(ctx.max() + 1) // 256) + page - 1) // page     # a seat holds a multiple of 256 positions
    pages = 1 + int(used.sum()) + 16
    ids = 1 + rng.permutation(pages - 1)
    table, at = np.full((len(ctx), width), -1, np.int32), 0
    for b in range(len(ctx)):
        table[b, :used[b]] = ids[at:at + used[b]]
        at += int(used[b])
    return torch.from_numpy(table).to(DEV), pages


def _stack(pages, case, g, s):
    """All layers' K and V in one tensor: bf16 [2 layers, pages, page, hkv, D], or the 8-bit pool's codes, a page's tokens of one
    head next to each other in memory, with their exponent bytes [2 layers, pages, hkv, page]."""
    n, p, h = 2 * case["layers"], case["page"], case["hkv"]
    if case["fp8"]:
        # 0x38..0x7e are 1 to 448: no code is a NaN, whose payload would not survive a comparison
        s.pool = torch.randint(0x38, 0x7f, (n, pages, h, p, D), generator=g, device=DEV, dtype=torch.uint8).view(E4).transpose(2, 3)
        s.scale = torch.randint(110, 130, (n, pages, h, p), generator=g, device=DEV, dtype=torch.uint8)
    else:
        s.pool = torch.empty((n, pages, p, h, D), dtype=BF, device=DEV)
        for i in range(n):
            s.pool[i].normal_(generator=g)
        s.scale = None
    s.caches = list(s.pool.unbind(0))
    s.scales = list(s.scale.unbind(0)) if case["fp8"] else []


def prepare(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    s = SimpleNamespace(case=case)
    page, hkv, kind = case["page"], case["hkv"], case["kind"]
    if kind in ("store", "read"):
        # Runs of consecutive positions in scattered pages; page 0 is the scratch page that no token has.
        T = case["tokens"]
        used = -(-T // page)
        pages = 1 + used + used // 8
        ids = 1 + rng.permutation(pages - 1)[:used]
        t = np.arange(T)
        slots = ids[t // page] * page + t % page
        slots[T - case["pads"]:] = -1
        s.slots = torch.from_numpy(slots.astype(np.int64)).to(DEV)
        s.kc, s.vc, s.ks, s.vs = _pool4(pages, case, g)
        if kind == "store":
            s.k = _keys((T, hkv, D), g)
            s.v = _values((T, 2 * hkv, D), g)[:, hkv:]     # a view of the projection's output
        return s
    if kind == "copy":
        n = case["pairs"]
        pages = 1 + 2 * n
        ids = 1 + rng.permutation(pages - 1)
        src = np.full(n, ids[0]) if case["fork"] else ids[:n]
        s.src, s.dst = (torch.from_numpy(x.astype(np.int32)).to(DEV) for x in (src, ids[n:2 * n]))
        _stack(pages, case, g, s)
        return s
    ctx = _contexts(case)
    s.table, pages = _tables(ctx, page, rng)
    if kind == "compact":
        _stack(pages, case, g, s)
        s.seqlens = torch.from_numpy(ctx).to(torch.int32).to(DEV)
        s.keep = torch.from_numpy(_kept(case)).to(DEV)
        return s
    B = case["rows"]
    s.longest = int(ctx.max())
    s.kc, s.vc, s.ks, s.vs = _pool4(pages, case, g)
    s.seqlens = torch.from_numpy(ctx - int(case["append"])).to(torch.int32).to(DEV)
    s.q = _keys((B, case["hq"], D), g)
    if case["append"]:
        s.k, s.v = _keys((B, hkv, D), g), _values((B, hkv, D), g)
        pos = s.seqlens.long()
        slot = s.table.long().gather(1, pos.clamp(min=0)[:, None] // page)[:, 0] * page + pos % page
        s.slots = torch.where(pos >= 0, slot, -1)
    return s


# ---------------------------------------------------------------------------------------------------- the plain form

def _value(codes, exps):
    """Packed codes [..., D / 2] and exponent bytes [..., D / 32] -> fp32 [..., D]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    m, e = (c & 1).float(), (c >> 1 & 3).int()
    a = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * _pow2(e - 1))
    x = torch.where(c >= 8, -a, a).unflatten(-1, (D // BLOCK, BLOCK))
    return (x * _pow2(exps.int() - 127)[..., None]).flatten(-2)


def _write(s, k, v, slots):
    """Rows k, v [T, hkv, D] into the pool's slots [T]; those below 0 put back what page 0 holds."""
    page = s.kc.shape[1]
    live = slots >= 0
    at = slots.clamp(min=0)
    p, o = at // page, at % page
    for x, pool, scale in ((k, s.kc, s.ks), (v, s.vc, s.vs)):
        c, e = _codes(x)
        pool[p, o] = torch.where(live[:, None, None], c, pool[p, o])
        scale[p, :, :, o] = torch.where(live[:, None, None], e, scale[p, :, :, o])


def _read(s, slots):
    page = s.kc.shape[1]
    live = (slots >= 0)[..., None, None]
    at = slots.clamp(min=0)
    p, o = at // page, at % page
    return [torch.where(live, _value(pool[p, o], scale[p, :, :, o]), 0.0) for pool, scale in ((s.kc, s.ks), (s.vc, s.vs))]


def _plain_attention(s, q, lens):
    """q [B, hq, D] over the first lens[b] tokens of each row."""
    B, hq, _ = q.shape
    page, hkv = s.kc.shape[1], s.kc.shape[2]
    at = torch.arange(s.longest, device=DEV)
    seen = at[None] < lens[:, None]
    slots = torch.where(seen, s.table.long()[:, at // page] * page + at % page, -1)
    k, v = _read(s, slots)                                                     # [B, L, hkv, D]
    x = q.float().view(B, hkv, hq // hkv, D)
    a = torch.matmul(x, k.permute(0, 2, 3, 1).contiguous()) * SCALE            # [B, hkv, G, L]
    a = torch.where(seen[:, None, None], a, -math.inf)
    m = a.amax(-1, keepdim=True)
    p = torch.exp(a - torch.where(torch.isfinite(m), m, 0.0))
    o = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous())
    o = torch.where((lens > 0)[:, None, None, None], o / p.sum(-1, keepdim=True), 0.0)
    return o.view(B, hq, D).to(BF)


def _bytes(pool):
    """The pool as elements that torch's indexing takes."""
    return pool.view(torch.uint8) if pool.dtype == E4 else pool


def _plain_compact(s):
    page = s.case["page"]
    at = torch.arange(s.keep.shape[1], device=DEV)
    kept = s.keep & (at < s.seqlens[:, None])
    n = kept.sum(1)
    order = torch.argsort((~kept).int(), dim=1, stable=True)
    src = torch.where(at < n[:, None], order, at)                              # what is behind the kept ones stays
    pages = s.table.long()[:, :-(-s.keep.shape[1] // page)].clamp(min=0)       # without a page: the scratch page, onto itself
    p0, o0 = pages.gather(1, src // page), src % page
    p1, o1 = pages[:, at // page], (at % page).expand_as(src)
    x = _bytes(s.pool)
    x[:, p1, o1] = x[:, p0, o0]
    if s.scale is not None:
        s.scale[:, p1, :, o1] = s.scale[:, p0, :, o0]
    return n.int()


def _plain(s):
    kind = s.case["kind"]
    if kind == "copy":
        src, dst = s.src.long(), s.dst.long()
        x = _bytes(s.pool)
        x[:, dst] = x[:, src]
        if s.scale is None:
            return {"pool": s.pool}
        s.scale[:, dst] = s.scale[:, src]
        return {"pool": s.pool, "scale": s.scale}
    if kind == "compact":
        n = _plain_compact(s)
        return {"pool": s.pool, "lengths": n, **({} if s.scale is None else {"scale": s.scale})}
    if kind == "store":
        _write(s, s.k, s.v, s.slots)
    if kind in ("store", "read"):
        k, v = _read(s, s.slots)
        return {"k": k.to(BF), "v": v.to(BF)}
    if not s.case["append"]:
        return {"out": _plain_attention(s, s.q, s.seqlens)}
    _write(s, s.k, s.v, s.slots)
    k, v = _read(s, s.slots)
    return {"out": _plain_attention(s, s.q, s.seqlens + 1), "k": k.to(BF), "v": v.to(BF)}


# ---------------------------------------------------------------------------------------------------- the operators

def _q3attn():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-tts-engine_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import q3attn
    return q3attn


def _operators(s):
    ops, kind = _q3attn(), s.case["kind"]
    if kind == "copy":
        ops.paged_copy(s.caches + s.scales, s.src, s.dst)
        return {"pool": s.pool, **({} if s.scale is None else {"scale": s.scale})}
    if kind == "compact":
        n = ops.paged_compact(s.caches, s.keep, s.seqlens, s.table, s.scales)
        return {"pool": s.pool, "lengths": n, **({} if s.scale is None else {"scale": s.scale})}
    if kind == "store":
        ops.paged_write_fp4(s.k, s.v, s.slots, s.kc, s.vc, s.ks, s.vs)
    if kind in ("store", "read"):
        k, v = ops.paged_read_fp4(s.kc, s.vc, s.ks, s.vs, s.slots)
        return {"k": k, "v": v}
    if not s.case["append"]:
        return {"out": ops.paged_decode_fp4(s.q, s.kc, s.vc, s.ks, s.vs, s.seqlens, s.table, SCALE)}
    out = ops.paged_decode_fp4_append(s.q, s.k, s.v, s.kc, s.vc, s.ks, s.vs, s.seqlens, s.table, SCALE)
    k, v = ops.paged_read_fp4(s.kc, s.vc, s.ks, s.vs, s.slots)
    return {"out": out, "k": k, "v": v}


def run(state):
    return _operators(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------- work, exact

def work(case):
    hkv, kind = case["hkv"], case["kind"]
    row4, row16 = hkv * 2 * (D // 2 + D // BLOCK), hkv * 2 * 2 * D             # a token's K and V in the 4-bit pool and in bf16
    if kind in ("store", "read"):
        live, T = case["tokens"] - case["pads"], case["tokens"]
        n_bytes = live * row4 + T * row16 + 8 * T
        return {"bytes": n_bytes + (live * row16 if kind == "store" else 0), "flops": 0}
    if kind in ("copy", "compact"):
        token = case["layers"] * hkv * 2 * (D + 1 if case["fp8"] else 2 * D)
    if kind == "copy":
        n = case["pairs"]
        return {"bytes": (n + (1 if case["fork"] else n)) * case["page"] * token + 8 * n, "flops": 0}
    ctx = _contexts(case)
    if kind == "compact":
        keep = _kept(case)
        stay = np.cumprod(keep, 1).sum()                                       # those in front of a row's first gap
        return {"bytes": 2 * int(keep.sum() - stay) * token + int(ctx.sum()) + 8 * len(ctx), "flops": 0}
    B, hq, live = case["rows"], case["hq"], case["rows"] - case["pads"]
    total = int(ctx.sum())
    n_bytes = total * row4 + 4 * D * hq * B + 4 * B + 4 * int((-(-ctx // case["page"])).sum())
    if case["append"]:
        n_bytes += live * row16 + B * (row16 + 8)   # the new rows are written, not read, in the pool; then they are read back
    return {"bytes": n_bytes, "flops": 4 * D * hq * total}


def _two(e):
    """2^e in 64 bits, from its bits."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_values(x):
    """What the 4-bit pool holds for rows x, from the definition in 64 bits."""
    x = x.double().unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True) / 7)
    e = torch.where(m > 0, torch.where(m > 0.5, e, e - 1), E_MIN).clamp(E_MIN, E_MAX)      # the least e with amax <= 7 * 2^e
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    y = (x / _two(e)).contiguous()
    a = y.abs().clamp(max=6)
    hi = torch.bucketize(a, grid)                                              # grid[hi - 1] < a <= grid[hi]
    lo = (hi - 1).clamp(min=0)
    down, up = a - grid[lo], grid[hi] - a
    near = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)   # a tie goes to the even code
    return (torch.copysign(grid[near], y) * _two(e)).flatten(-2)


def _exact_pool(codes, exps):
    """Packed codes [..., D / 2] and exponents [..., D / 32] as values in 64 bits."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=codes.device)
    x = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).flatten(-2)
    return x * _two(exps.int() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    kind, page = case["kind"], case["page"]
    if kind in ("copy", "compact"):
        return None                                                            # values are moved, none is computed
    s = prepare(case, seed)
    if kind == "store":
        live = (s.slots >= 0)[:, None, None]
        return {n: torch.where(live, _exact_values(x), 0.0) for n, x in (("k", s.k), ("v", s.v))}
    if kind == "read":
        live = (s.slots >= 0)[:, None, None]
        pg, off = s.slots.clamp(min=0) // page, s.slots.clamp(min=0) % page
        return {n: torch.where(live, _exact_pool(pool[pg, off], scale[pg, :, :, off]), 0.0)
                for n, pool, scale in (("k", s.kc, s.ks), ("v", s.vc, s.vs))}
    B, hq, hkv = case["rows"], case["hq"], case["hkv"]
    new = {}
    if case["append"]:
        live = (s.slots >= 0)[:, None, None]
        new = {n: torch.where(live, _exact_values(x), 0.0) for n, x in (("k", s.k), ("v", s.v))}
    q, out = s.q.double(), torch.zeros((B, hq, D), dtype=torch.float64, device=DEV)
    for b, n in enumerate(s.seqlens.tolist()):
        if n < 0 or (n == 0 and not case["append"]):
            continue
        ids = s.table[b, :-(-n // page)].long()
        k, v = (_exact_pool(pool[ids], scale[ids].permute(0, 3, 1, 2)).reshape(-1, hkv, D)[:n]
                for pool, scale in ((s.kc, s.ks), (s.vc, s.vs)))
        if case["append"]:
            k, v = torch.cat([k, new["k"][b][None]]), torch.cat([v, new["v"][b][None]])
        for h in range(hkv):
            x = q[b, h * (hq // hkv):(h + 1) * (hq // hkv)]
            out[b, h * (hq // hkv):(h + 1) * (hq // hkv)] = (x @ k[:, h].T * SCALE).softmax(-1) @ v[:, h]
    return {"out": out, **new}
