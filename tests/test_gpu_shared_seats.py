"""Seats that share pages, from the pool to the kernels: a prompt is forked, the forks go on by tokens of their own, some let go of tokens,
are cut back and go on, the pages are moved together.  After every stage each seat's tokens read back, and attention over them, have the
bits of a pool whose seats share nothing and whose contents were written at once; over the bf16, the 8-bit and the 4-bit pool."""
import numpy as np
import pytest
import torch

import q3attn
from q3attn.pages import PagePool

pytestmark = pytest.mark.gpu

LAYERS, SEATS, WIDTH, PAGE, HKV, HQ, SCALE = 2, 4, 10, 16, 2, 4, 128 ** -0.5


class Stack:
    """All layers' pools of one kind."""

    def __init__(self, kind, pages, dev):
        self.kind, self.dev = kind, dev
        if kind == "bf16":
            self.layers = [[torch.zeros((pages, PAGE, HKV, 128), dtype=torch.bfloat16, device=dev) for _ in range(2)] for _ in range(LAYERS)]
        else:
            make = q3attn.fp8_cache if kind == "fp8" else q3attn.fp4_cache
            self.layers = [list(make(pages, PAGE, HKV, device=dev)) for _ in range(LAYERS)]

    @property
    def caches(self):
        return [t for x in self.layers for t in x[:2]]

    @property
    def scales(self):
        return [t for x in self.layers for t in x[2:]]

    def _op(self, name):
        return getattr(q3attn, name.replace("*", self.kind))

    def write(self, i, k, v, slots):
        x = self.layers[i]
        if self.kind == "bf16":
            x[0].view(-1, HKV, 128).index_copy_(0, slots, k)
            x[1].view(-1, HKV, 128).index_copy_(0, slots, v)
        else:
            self._op("paged_write_*")(k, v, slots, *x)

    def read(self, i, slots):
        x = self.layers[i]
        if self.kind == "bf16":
            return [t.view(-1, HKV, 128)[slots] for t in x]
        return self._op("paged_read_*")(*x, slots)

    def decode(self, i, q, ctx, table):
        return self._op("paged_decode" if self.kind == "bf16" else "paged_decode_*")(q, *self.layers[i], ctx, table, SCALE)

    def append(self, i, q, k, v, ctx, table):
        return self._op("paged_decode_append" if self.kind == "bf16" else "paged_decode_*_append")(q, k, v, *self.layers[i], ctx, table, SCALE)


class Server:
    def __init__(self, kind, dev, checks):
        self.pool = PagePool(num_pages=40, max_seats=SEATS, max_pages_per_seat=WIDTH, page_size=PAGE, device=dev)
        self.stack, self.own = Stack(kind, 40, dev), Stack(kind, SEATS * WIDTH, dev)
        self.own_table = torch.arange(SEATS * WIDTH, dtype=torch.int32, device=dev).view(SEATS, WIDTH)
        self.all = torch.arange(SEATS, device=dev)
        self.g, self.dev, self.checks = torch.Generator(device=dev), dev, checks
        self.g.manual_seed(3)
        none = torch.zeros((0, HKV, 128), dtype=torch.bfloat16, device=dev)
        self.hist = [[[none, none] for _ in range(LAYERS)] for _ in range(SEATS)]     # every seat's K and V rows, a layer each

    def rand(self, *shape):
        return torch.randn(shape, generator=self.g, device=self.dev).to(torch.bfloat16)

    def length(self, s):
        return len(self.hist[s][0][0])

    def ctx(self, seats=range(SEATS)):
        return torch.tensor([self.length(s) for s in seats], dtype=torch.int32, device=self.dev)

    def copy(self, pairs):
        q3attn.paged_copy(self.stack.caches + self.stack.scales, *pairs)

    def note(self, s, i, k, v):
        self.hist[s][i] = [torch.cat([old, new]) for old, new in zip(self.hist[s][i], (k, v))]

    def prompt(self, s, n):
        first = self.length(s)
        self.pool.grow(s, first + n)
        pos = torch.arange(first, first + n, device=self.dev)
        slots = self.pool.slot(torch.full_like(pos, s), pos)
        for i in range(LAYERS):
            k, v = self.rand(n, HKV, 128), self.rand(n, HKV, 128)
            self.stack.write(i, k, v, slots)
            self.note(s, i, k, v)

    def step(self, seats):
        """One token more for each of ``seats``, in one call a layer."""
        self.pool.grow(seats, [self.length(s) + 1 for s in seats])
        ctx = torch.tensor([self.length(s) if s in seats else -1 for s in range(SEATS)], dtype=torch.int32, device=self.dev)
        if self.checks:
            self.fill_own()
        for i in range(LAYERS):
            q, k, v = self.rand(SEATS, HQ, 128), self.rand(SEATS, HKV, 128), self.rand(SEATS, HKV, 128)
            out = self.stack.append(i, q, k, v, ctx, self.pool.block_table(self.all))
            if self.checks:
                assert torch.equal(out, self.own.append(i, q, k, v, ctx, self.own_table))
            for s in seats:
                self.note(s, i, k[s:s + 1], v[s:s + 1])
        self.check()

    def drop(self, seats, keep):
        """The seats let go of the tokens that ``keep`` (a mask a seat) names."""
        first = [int(np.argmin(m.numpy())) for m in keep]
        self.copy(self.pool.unshare(seats, first))
        mask = torch.zeros((len(seats), max(len(m) for m in keep)), dtype=torch.bool)
        for row, m in zip(mask, keep):
            row[:len(m)] = m
        table = self.pool.block_table(torch.tensor(seats, device=self.dev))
        new = q3attn.paged_compact(self.stack.caches, mask.to(self.dev), self.ctx(seats), table, self.stack.scales)
        for s, m in zip(seats, keep):
            self.hist[s] = [[x[m.to(self.dev)] for x in kv] for kv in self.hist[s]]
        assert new.tolist() == [self.length(s) for s in seats]
        self.pool.truncate(seats, new.tolist())
        self.check()

    def fill_own(self):
        for s in range(SEATS):
            slots = s * WIDTH * PAGE + torch.arange(self.length(s), device=self.dev)
            for i in range(LAYERS):
                self.own.write(i, *self.hist[s][i], slots)

    def check(self, always=False):
        if not (self.checks or always):
            return
        self.pool.check()
        self.fill_own()
        ctx, table = self.ctx(), self.pool.block_table(self.all)
        for i in range(LAYERS):
            for s in range(SEATS):
                pos = torch.arange(self.length(s), device=self.dev)
                for a, b in zip(self.stack.read(i, self.pool.slot(torch.full_like(pos, s), pos)), self.own.read(i, s * WIDTH * PAGE + pos)):
                    assert torch.equal(a, b), (s, i)
            q = self.rand(SEATS, HQ, 128)
            out = self.stack.decode(i, q, ctx, table)
            assert torch.equal(out, self.own.decode(i, q, ctx, self.own_table)), i
            assert torch.isfinite(out.float()).all() and bool(out[ctx > 0].any()) and not out[ctx == 0].any()

    def fork(self, src, seats, length):
        self.copy(self.pool.fork(src, seats, length))
        for s in seats:
            self.hist[s] = [[x[:length] for x in kv] for kv in self.hist[src]]
        self.check()

    def release(self, s):
        self.pool.release(s)
        self.hist[s] = [[x[:0] for x in kv] for kv in self.hist[s]]
        self.check()

    def truncate(self, s, length):
        self.pool.truncate(s, length)
        self.hist[s] = [[x[:length] for x in kv] for kv in self.hist[s]]
        self.check()
        self.copy(self.pool.unshare(s, length))              # its last page may be shared, and is written next
        self.check()

    def defragment(self):
        used = len({p for s in range(SEATS) for p in self.pool.pages_of(s)})
        src, dst = self.pool.defragment()
        self.copy((src, dst))
        self.check()
        assert max(p for s in range(SEATS) for p in self.pool.pages_of(s)) == used
        return len(src)


@pytest.mark.parametrize("kind", ["bf16", "fp8", "fp4"])
@pytest.mark.parametrize("checks,side", [(True, False), (True, True), (False, False), (False, True)])
def test_forked_compacted_and_moved_seats(cuda_device, kind, checks, side):
    """``checks`` False: nothing waits for the GPU between the stages but where a program does (the lengths after a compaction)."""
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        m = Server(kind, cuda_device, checks)
        g = torch.Generator().manual_seed(5)
        m.prompt(0, 77)
        m.check()
        m.fork(0, [1, 2], 77)                                # four pages shared, the last one copied for each
        assert m.pool.pages_of(1)[:4] == m.pool.pages_of(0)[:4] and len(set(m.pool.pages_of(s)[4] for s in range(3))) == 3
        for _ in range(5):                                   # over the end of the copied page
            m.step([0, 1, 2])
        masks = [torch.rand(82, generator=g) < 0.6 for _ in range(2)]
        masks[0][:30], masks[0][30], masks[1][0] = True, False, False
        m.drop([1, 2], masks)                                # seat 1's first page stays shared, nothing of seat 2
        assert m.pool.pages_of(1)[0] == m.pool.pages_of(0)[0] and not set(m.pool.pages_of(2)) & set(m.pool.pages_of(0))
        m.step([1, 2])
        n = m.length(1) - 3
        m.fork(1, [3], n)
        m.release(0)                                         # shared pages outlive it
        m.step([1, 2, 3])
        m.truncate(3, 20)                                    # inside a page that seat 1 holds too
        assert m.pool.pages_of(3)[0] == m.pool.pages_of(1)[0] and m.pool.pages_of(3)[1] != m.pool.pages_of(1)[1]
        for _ in range(3):
            m.step([3, 2])
        assert m.defragment() > 0
        m.prompt(0, 50)                                      # in pages that others have left
        m.step([0, 1, 2, 3])
        m.check(always=True)
    stream.synchronize()
