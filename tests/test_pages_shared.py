"""CPU tests of the page pool's shared pages: forks, pages of one's own again, truncation and moving the pages together, against a
model that holds every seat's tokens."""
import numpy as np
import pytest
import torch

from q3attn.pages import PagePool, PoolExhausted


class Model:
    """A pool with contents: one number a token, copied as the pairs say."""

    def __init__(self, **kw):
        self.pool = PagePool(device="cpu", **kw)
        self.mem = np.zeros((self.pool.num_pages, self.pool.page_size), np.int64)
        self.tokens = [[] for _ in range(self.pool.max_seats)]
        self.next = 1

    def copy(self, pairs):
        src, dst = (x.tolist() for x in pairs)
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        for p, q in zip(src, dst):
            self.mem[q] = self.mem[p]

    def write(self, seat, first):
        """Positions ``first`` on of the seat get new numbers."""
        for t in range(first, len(self.tokens[seat])):
            self.tokens[seat][t] = self.next
            page = int(self.pool.table[seat, t // self.pool.page_size])
            self.mem[page, t % self.pool.page_size] = self.next
            self.next += 1

    def check(self):
        self.pool.check()
        for s, want in enumerate(self.tokens):
            page = self.pool.table[s].numpy()
            assert [int(self.mem[page[t // self.pool.page_size], t % self.pool.page_size]) for t in range(len(want))] == want


def test_random_sequences_keep_every_seats_tokens():
    rng = np.random.default_rng(0)
    m = Model(num_pages=120, max_seats=10, max_pages_per_seat=9, page_size=16)
    did = {}
    for _ in range(1500):
        s, act = int(rng.integers(10)), rng.choice(["grow", "grow", "grow", "fork", "release", "truncate", "unshare", "defragment"])
        n = len(m.tokens[s])
        try:
            if act == "grow":
                to = min(n + int(rng.integers(1, 30)), m.pool.seat_len)
                m.copy(m.pool.unshare(s, n))                               # a truncated seat's last page may be shared
                m.pool.grow(s, to)
                m.tokens[s] += [0] * (to - n)
                m.write(s, n)
            elif act == "fork":
                to = [x for x in rng.permutation(10)[:3].tolist() if x != s and not m.tokens[x] and not m.pool.pages_of(x)]
                length = int(rng.integers(0, n + 1))
                m.copy(m.pool.fork(s, to, length))
                for x in to:
                    m.tokens[x] = m.tokens[s][:length]
            elif act == "release":
                m.pool.release(s)
                m.tokens[s] = []
            elif act == "truncate":
                to = int(rng.integers(0, n + 1))
                m.pool.truncate(s, to)
                m.tokens[s] = m.tokens[s][:to]
            elif act == "unshare":
                first = int(rng.integers(0, n + 1))
                m.copy(m.pool.unshare(s, first))
                m.write(s, first)
            else:
                m.copy(m.pool.defragment())
            did[act] = did.get(act, 0) + 1
        except PoolExhausted:
            did["exhausted"] = did.get("exhausted", 0) + 1
        m.check()
    assert min(did.values()) > 20 and len(did) >= 6, did


def test_fork_shares_full_pages_and_copies_the_last():
    pool = PagePool(num_pages=20, max_seats=4, max_pages_per_seat=6, device="cpu")
    pool.grow(0, 77)                                                       # the voice prefix: 4 pages and 13 tokens
    src, dst = pool.fork(0, [1, 2], 77)
    assert src.dtype == dst.dtype == torch.int32 and src.tolist() == [pool.pages_of(0)[4]] * 2
    assert pool.pages_of(1)[:4] == pool.pages_of(2)[:4] == pool.pages_of(0)[:4] and pool.pages_of(1)[4:] == [dst[0]] and dst[0] != dst[1]
    assert pool.free_pages == 20 - 1 - 5 - 2
    pool.release(0)
    assert pool.free_pages == 20 - 1 - 4 - 2                               # only the page that seat 0 alone held
    src, dst = pool.fork(1, 0, 64)
    assert len(src) == len(dst) == 0 and pool.pages_of(0) == pool.pages_of(1)[:4]
    pool.grow(0, 70)
    pool.check()
    pool.release([0, 1, 2])
    assert pool.free_pages == 19
    pool.check()


def test_unshare_leaves_the_last_holder_its_page():
    pool = PagePool(num_pages=20, max_seats=3, max_pages_per_seat=4, device="cpu")
    pool.grow(0, 64)
    pool.fork(0, [1, 2], 64)
    old = pool.pages_of(0)
    src, dst = pool.unshare([0, 1], [32, 16])
    assert pool.pages_of(0)[:2] == old[:2] and pool.pages_of(1)[0] == old[0] and pool.pages_of(2) == old
    assert src.tolist() == old[2:] + old[1:] and len(set(dst.tolist())) == 5
    pool.check()
    assert [len(x) for x in pool.unshare(2, 32)] == [0, 0]                 # pages 2 and 3 are its own by now
    src, dst = pool.unshare([0, 1, 2])                                     # page 0 thrice, page 1 twice: the last one keeps each
    assert sorted(src.tolist()) == sorted([old[0], old[0], old[1]]) and pool.pages_of(2) == old
    pool.check()


def test_defragment_moves_shared_pages_once():
    pool = PagePool(num_pages=30, max_seats=4, max_pages_per_seat=6, device="cpu")
    pool.grow([0, 1], [96, 96])
    pool.fork(1, 2, 96)
    pool.release(0)
    src, dst = pool.defragment()
    assert sorted(dst.tolist()) == [1, 2, 3, 4, 5, 6] and sorted(src.tolist()) == [7, 8, 9, 10, 11, 12]
    assert pool.pages_of(1) == pool.pages_of(2) and sorted(pool.pages_of(1)) == [1, 2, 3, 4, 5, 6]
    pool.check()
    assert [len(x) for x in pool.defragment()] == [0, 0]
    pool.grow(0, 16)
    assert pool.pages_of(0) == [7]


def test_all_or_nothing_and_refusals():
    pool = PagePool(num_pages=7, max_seats=5, max_pages_per_seat=4, device="cpu")
    pool.grow([0, 1], [20, 40])                                            # 2 + 3 pages, 1 left
    before = pool.table.clone()
    with pytest.raises(PoolExhausted):
        pool.fork(0, [2, 3], 20)
    assert torch.equal(pool.table, before) and not pool.pages_of(2)
    pool.fork(0, 2, 16)
    pool.fork(0, 3, 16)
    before = pool.table.clone()
    with pytest.raises(PoolExhausted):
        pool.unshare([0, 2, 3])
    assert torch.equal(pool.table, before)
    pool.check()
    for bad in (lambda: pool.fork(0, 1, 16), lambda: pool.fork(0, [4, 4], 16), lambda: pool.fork(0, 4, 33), lambda: pool.fork(0, 4, -1),
                lambda: pool.unshare([0, 0]), lambda: pool.truncate([0, 1], [3])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: pool.fork(5, 4, 0), lambda: pool.fork(0, 5, 0), lambda: pool.unshare(-1), lambda: pool.truncate(5, 0)):
        with pytest.raises(IndexError):
            bad()
    assert torch.equal(pool.table, before)
    pool.check()
