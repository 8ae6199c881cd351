"""Paged KV pool bookkeeping: 16-token pages handed out to seats from a free list.

The reference gives every seat a fixed, contiguous slice of the KV pool (pages of 256 positions and an identity
``seat_pages`` table, engine/talker.py:23-31, 42; append slot ``seat * seat_len + pos``, engine/talker.py:109).
Here the pool is shared: a seat owns only the pages its tokens occupy, taken from a free list as it grows and
returned when it is released, so memory follows the live contexts instead of ``n_seats * seat_len``.

* ``table`` is a device-resident ``[max_seats + 1, max_pages_per_seat]`` int32 block table (row ``max_seats`` is the
  scratch seat that padded rows use, engine/talker.py:27, 110-111; all its entries point at the reserved scratch
  page).  Unallocated entries hold -1 (the decode kernels treat out-of-range page ids as "no tokens").
* ``grow`` / ``release`` run on the host between frames and push only the changed table entries to the device
  (one indexed write per call).
* ``block_table(seat)`` and ``slot(seat, pos)`` are plain tensor ops on device tensors, so a captured frame graph
  computes its rows' tables and append slots from the device-resident seat ids and positions, as
  ``Talker._frame`` does (engine/talker.py:107-112).

* Seats may share pages: ``fork`` gives seats the pages of another one's first tokens (samples of one prompt, the voice prefix
  that the reference copies into every seat, engine/arrivals.py:118-145), ``unshare`` gives a seat pages of its own again before
  tokens in them are rewritten, and a page is free when its last seat lets go of it.  ``truncate`` frees the pages behind a row's
  end, ``defragment`` moves the used pages together.  Where contents have to follow, these return the page pairs for
  ``q3attn.paged_copy``.  The pool holds neither side of a pair until then: a source page may be free already, and the next call may
  hand it out.  So each call's pairs are copied by a ``paged_copy`` of their own (pairs of two calls may chain, one's destination the
  other's source, which one copy does not follow), on the stream that decodes, and before the pool's next call.

The pool tensors themselves (``[num_pages, page_size, kv_heads, head_dim]`` per layer) are the caller's; this class
only decides which page ids hold which seat's tokens.
"""
from __future__ import annotations

import numpy as np
import torch


class PoolExhausted(RuntimeError):
    """No free page is left for a seat that must grow."""


class PagePool:
    SCRATCH_PAGE = 0

    def __init__(self, num_pages: int, max_seats: int, max_pages_per_seat: int, page_size: int = 16,
                 device="cuda"):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} must be a power of two >= 16")
        if num_pages < 2 or max_seats < 1 or max_pages_per_seat < 1:
            raise ValueError("need num_pages >= 2 (one is the scratch page), max_seats >= 1, max_pages_per_seat >= 1")
        self.num_pages, self.max_seats, self.max_pages, self.page_size = num_pages, max_seats, max_pages_per_seat, page_size
        self.scratch_seat = max_seats
        self.device = torch.device(device)
        # Free list as a stack; low page ids are handed out first.
        self._free = list(range(num_pages - 1, self.SCRATCH_PAGE, -1))
        self._pages = [[] for _ in range(max_seats)]          # host copy of each seat's page list
        self._refs = [0] * num_pages                          # seats that hold the page
        host = np.full((max_seats + 1, max_pages_per_seat), -1, np.int32)
        host[max_seats, :] = self.SCRATCH_PAGE
        self.table = torch.from_numpy(host).to(self.device)

    # ------------------------------------------------------------------ host-side bookkeeping
    @property
    def seat_len(self) -> int:
        """Positions one seat can hold."""
        return self.max_pages * self.page_size

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages_of(self, seat: int) -> list:
        return list(self._pages[seat])

    def capacity(self, seat: int) -> int:
        """Positions seat ``seat`` can hold with its current pages."""
        return len(self._pages[seat]) * self.page_size

    def grow(self, seats, lengths) -> None:
        """Give each seat enough pages for ``length`` positions (0..length-1).  All-or-nothing: raises
        PoolExhausted (changing nothing) when the free list cannot cover the request."""
        seats = [int(s) for s in np.atleast_1d(seats)]
        lengths = [int(n) for n in np.atleast_1d(lengths)]
        if len(seats) != len(lengths):
            raise ValueError("seats and lengths differ in length")
        need = {}
        for s, n in zip(seats, lengths):
            if not 0 <= s < self.max_seats:
                raise IndexError(f"seat {s} outside [0, {self.max_seats})")
            if n > self.seat_len:
                raise ValueError(f"seat {s}: length {n} exceeds {self.seat_len} positions")
            want = -(-max(n, 0) // self.page_size)
            need[s] = max(need.get(s, 0), want)
        extra = sum(max(0, w - len(self._pages[s])) for s, w in need.items())
        if extra > len(self._free):
            raise PoolExhausted(f"{extra} pages needed, {len(self._free)} free")
        rows, cols, vals = [], [], []
        for s, w in need.items():
            pl = self._pages[s]
            while len(pl) < w:
                p = self._take()
                rows.append(s)
                cols.append(len(pl))
                vals.append(p)
                pl.append(p)
        self._write(rows, cols, vals)

    def _take(self) -> int:
        p = self._free.pop()
        self._refs[p] = 1
        return p

    def _drop(self, pages) -> None:
        """One seat lets go of ``pages``; those that no other seat holds are free."""
        for p in pages:
            self._refs[p] -= 1
        self._free.extend(p for p in reversed(pages) if self._refs[p] == 0)

    def _seat(self, seat) -> int:
        seat = int(seat)
        if not 0 <= seat < self.max_seats:
            raise IndexError(f"seat {seat} outside [0, {self.max_seats})")
        return seat

    def _pairs(self, src, dst):
        pair = torch.tensor([src, dst], dtype=torch.int32).reshape(2, -1)
        if self.device.type != "cpu":
            pair = pair.pin_memory().to(self.device, non_blocking=True)
        return pair[0], pair[1]

    def release(self, seats) -> None:
        """Return the seats' pages to the free list and clear their table rows."""
        rows, cols, vals = [], [], []
        for s in (int(x) for x in np.atleast_1d(seats)):
            if not 0 <= s < self.max_seats:
                raise IndexError(f"seat {s} outside [0, {self.max_seats})")
            pl = self._pages[s]
            for i in range(len(pl)):
                rows.append(s)
                cols.append(i)
                vals.append(-1)
            self._drop(pl)
            self._pages[s] = []
        self._write(rows, cols, vals)

    def truncate(self, seats, lengths) -> None:
        """Free the pages that each seat holds behind its first ``length`` positions (after ``paged_compact``, or when drafted
        tokens are given up).  A last page that is cut inside may be shared: ``unshare(seat, length)`` before the seat writes on."""
        seats, lengths = [self._seat(s) for s in np.atleast_1d(seats)], [int(n) for n in np.atleast_1d(lengths)]
        if len(seats) != len(lengths):
            raise ValueError("seats and lengths differ in length")
        rows, cols, vals = [], [], []
        for s, n in zip(seats, lengths):
            stay = -(-max(n, 0) // self.page_size)
            gone = self._pages[s][stay:]
            for i in range(len(gone)):
                rows.append(s)
                cols.append(stay + i)
                vals.append(-1)
            self._drop(gone)
            self._pages[s] = self._pages[s][:stay]
        self._write(rows, cols, vals)

    def fork(self, src, seats, length: int):
        """Give each of ``seats``, which hold nothing yet, the first ``length`` positions of seat ``src``: its full pages, shared, and a
        page of their own for the tokens of a last, partly filled one, which they go on writing.  Returns (src, dst), int32 [pairs]
        on the pool's device: the pages that ``q3attn.paged_copy`` has to copy in every cache (none if ``length`` ends with a page).
        The copy has to be enqueued before the pool's next call (which may hand out the source page, if its seat is released), before
        the source page is written again and before anything reads the forks; pairs of several calls are not to be joined into one
        copy.  All-or-nothing: raises PoolExhausted (changing nothing) when the free list cannot cover them."""
        src, seats, length = self._seat(src), [self._seat(s) for s in np.atleast_1d(seats)], int(length)
        if not 0 <= length <= self.capacity(src):
            raise ValueError(f"seat {src} holds {self.capacity(src)} positions, not {length}")
        if len(set(seats)) != len(seats) or any(self._pages[s] for s in seats):
            raise ValueError("forks need seats that hold no pages, each named once")
        full, part = divmod(length, self.page_size)
        need = len(seats) if part else 0
        if need > len(self._free):
            raise PoolExhausted(f"{need} pages needed, {len(self._free)} free")
        shared = self._pages[src][:full]
        rows, cols, vals, dst = [], [], [], []
        for s in seats:
            for p in shared:
                self._refs[p] += 1
            pl = list(shared)
            if part:
                dst.append(self._take())
                pl.append(dst[-1])
            rows += [s] * len(pl)
            cols += range(len(pl))
            vals += pl
            self._pages[s] = pl
        self._write(rows, cols, vals)
        return self._pairs([self._pages[src][full]] * len(dst) if part else [], dst)

    def unshare(self, seats, first=0):
        """Give each seat pages of its own from the one that holds position ``first`` on (a number, or one a seat), in place of those
        that it shares: before tokens in them are rewritten (``paged_compact``).  Returns the pairs to copy, under the same conditions,
        and raises PoolExhausted, as ``fork``."""
        seats = [self._seat(s) for s in np.atleast_1d(seats)]
        firsts = [max(0, int(n)) // self.page_size for n in np.broadcast_to(first, (len(seats),))]
        if len(set(seats)) != len(seats):
            raise ValueError("each seat may be named once")
        left, todo = {}, []                                   # a page's last holder among them keeps it, if it is nobody else's
        for s, i0 in zip(seats, firsts):
            for i in range(i0, len(self._pages[s])):
                p = self._pages[s][i]
                if left.setdefault(p, self._refs[p]) > 1:
                    left[p] -= 1
                    todo.append((s, i, p))
        if len(todo) > len(self._free):
            raise PoolExhausted(f"{len(todo)} pages needed, {len(self._free)} free")
        dst = []
        for s, i, p in todo:
            self._refs[p] -= 1
            dst.append(self._take())
            self._pages[s][i] = dst[-1]
        self._write([s for s, _, _ in todo], [i for _, i, _ in todo], dst)
        return self._pairs([p for _, _, p in todo], dst)

    def defragment(self):
        """Move the used pages to the lowest ids, so that the pool's end is free.  Returns the pairs to copy, under the same conditions as
        ``fork``'s: their sources are free afterwards."""
        used = sorted(p for p in range(self.num_pages) if self._refs[p] > 0)
        src = [p for p in used if p > len(used)]              # page 0 is the scratch page
        dst = sorted(p for p in self._free if p <= len(used))
        new = dict(zip(src, dst))
        rows, cols, vals = [], [], []
        for s, pl in enumerate(self._pages):
            for i, p in enumerate(pl):
                if p in new:
                    pl[i] = new[p]
                    rows.append(s)
                    cols.append(i)
                    vals.append(new[p])
        for p, q in new.items():
            self._refs[q], self._refs[p] = self._refs[p], 0
        self._free = list(range(self.num_pages - 1, len(used), -1))
        self._write(rows, cols, vals)
        return self._pairs(src, dst)

    def _write(self, rows, cols, vals) -> None:
        if not rows:
            return
        idx_r = torch.tensor(rows, dtype=torch.long)
        idx_c = torch.tensor(cols, dtype=torch.long)
        v = torch.tensor(vals, dtype=torch.int32)
        if self.device.type != "cpu":
            idx_r, idx_c, v = (t.pin_memory().to(self.device, non_blocking=True) for t in (idx_r, idx_c, v))
        self.table.index_put_((idx_r, idx_c), v)

    def check(self) -> None:
        """Invariant check (tests and debugging): every page is free, scratch, or held by as many seats as are counted for it
        (in none of them twice), and the device table matches the host lists."""
        held = [0] * self.num_pages
        for pl in self._pages:
            for p in pl:
                held[p] += 1
        owned = [p for p in range(self.num_pages) if held[p] > 0]
        all_ids = owned + self._free + [self.SCRATCH_PAGE]
        if sorted(all_ids) != list(range(self.num_pages)) or held != self._refs or any(len(set(pl)) != len(pl) for pl in self._pages):
            raise AssertionError("page accounting broken: pages lost or handed out twice")
        host = self.table.cpu().numpy()
        for s, pl in enumerate(self._pages):
            row = host[s]
            if list(row[: len(pl)]) != pl or (row[len(pl):] != -1).any():
                raise AssertionError(f"device table row {s} differs from the host page list")

    # ------------------------------------------------------------------ device-side views (graph-capturable)
    def block_table(self, seat: torch.Tensor) -> torch.Tensor:
        """Rows of the block table for a batch of seat ids (int64 device tensor) -> [B, max_pages] int32."""
        return self.table.index_select(0, seat)

    def slot(self, seat: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        """Flat append slot (page * page_size + offset) of position ``pos`` of each seat, int64: the index the
        reference computes as ``seat * seat_len + pos`` (engine/talker.py:109) for its identity table."""
        page = self.table[seat, torch.div(pos, self.page_size, rounding_mode="floor")].long()
        return page * self.page_size + pos % self.page_size
