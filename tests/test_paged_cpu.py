"""Paged caches without a GPU: the page table against a plain model of what every sequence holds, the
4-bit weight layout, and the rings of the paged attention kernels as a protocol."""
import random

import numpy as np
import pytest

from mira_b200 import kernels as K
from mira_b200.paged import OutOfPages, PageTable


class Model:
    """Pages with contents (the token written at each slot) and, beside them, every sequence's tokens."""

    def __init__(self, num_pages, page_size, batch, max_pages):
        self.t = PageTable(num_pages, page_size, batch, max_pages)
        self.pages = [[None] * page_size for _ in range(num_pages)]
        self.tokens = {}
        self.next = 0

    def copy(self, src, dst):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        for a, b in zip(src, dst):
            self.pages[b] = list(self.pages[a])

    def extend(self, slot, n):
        before = len(self.tokens[slot])
        self.t.extend(slot, n)
        for i in range(before, before + n):
            page = self.t.table[slot, i // self.t.page_size]
            assert self.t.holders[page] == 1, "rows are appended to a shared page"
            self.pages[page][i % self.t.page_size] = self.next
            self.tokens[slot].append(self.next)
            self.next += 1

    def check(self):
        t = self.t
        count = np.zeros(t.num_pages, int)
        for slot in range(t.batch):
            assert bool(t.live[slot]) == (slot in self.tokens)
            assert t.lengths[slot] == len(self.tokens.get(slot, []))
            n = -(-int(t.lengths[slot]) // t.page_size)
            assert (t.table[slot, n:] == -1).all()
            for i, tok in enumerate(self.tokens.get(slot, [])):
                page = t.table[slot, i // t.page_size]
                if page >= 0:
                    assert self.pages[page][i % t.page_size] == tok
            for page in t.table[slot, :n]:
                if page >= 0:
                    count[page] += 1
        assert np.array_equal(count, t.holders)
        assert sorted(t._free) == np.flatnonzero(count == 0).tolist()


@pytest.mark.parametrize("seed", range(8))
def test_page_table_keeps_every_sequence(seed):
    rng = random.Random(seed)
    m = Model(num_pages=rng.choice([7, 40, 200]), page_size=rng.choice([1, 3, 16]), batch=rng.choice([2, 9]), max_pages=30)
    for _ in range(400):
        what = rng.choice(["open", "extend", "extend", "extend", "fork", "close", "compact", "trim"])
        some = rng.choice(sorted(m.tokens)) if m.tokens else None
        before = (m.t.table.copy(), m.t.lengths.copy(), m.t.holders.copy(), m.t.live.copy())
        try:
            if what == "open":
                m.tokens[m.t.open()] = []
            elif some is None:
                continue
            elif what == "extend":
                m.extend(some, rng.choice([0, 1, 1, 2, 20]))
            elif what == "fork":
                other, src, dst = m.t.fork(some)
                m.copy(src, dst)
                m.tokens[other] = list(m.tokens[some])
            elif what == "close":
                m.t.close(some)
                del m.tokens[some]
            elif what == "trim" and rng.random() < 0.3:
                window, sinks = rng.choice([1, 5, 40]), rng.choice([0, 1, 4])
                m.t.trim(some, window, sinks)
                # what the window and the sinks see is still there
                n = len(m.tokens[some])
                for i in list(range(min(sinks, n))) + list(range(max(0, n - window), n)):
                    assert m.t.table[some, i // m.t.page_size] >= 0 or i < 0 or before[0][some, i // m.t.page_size] < 0
            elif what == "compact":
                src, dst = m.t.compact()
                m.copy(src, dst)
                assert (m.t.holders[: m.t.used_pages()] > 0).all() and (m.t.holders[m.t.used_pages():] == 0).all()
        except OutOfPages:
            after = (m.t.table, m.t.lengths, m.t.holders, m.t.live)
            assert all(np.array_equal(a, b) for a, b in zip(before, after))
        m.check()


def test_fork_shares_full_pages_and_copies_the_last():
    t = PageTable(10, 4, 3, 8)
    a = t.open()
    t.extend(a, 10)
    b, src, dst = t.fork(a)
    assert src == [2] and dst == [3] and t.holders.tolist()[:4] == [2, 2, 1, 1]
    t.close(a)
    assert t.holders.tolist()[:4] == [1, 1, 0, 1] and t.free_pages() == 7
    c, src, dst = t.fork(b)
    t.close(c)
    assert t.used_pages() == 3
    full = t.open()
    t.extend(full, 8)
    assert t.fork(full)[1:] == ([], [])


def test_page_table_refusals():
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)):
        with pytest.raises(ValueError):
            PageTable(*bad)
    t = PageTable(4, 2, 2, 3)
    for call in (lambda: t.extend(0), lambda: t.fork(0), lambda: t.close(0), lambda: t.close(-1), lambda: t.trim(1, 3), lambda: t.extend(7)):
        with pytest.raises(ValueError):
            call()
    a = t.open()
    with pytest.raises(ValueError):
        t.extend(a, -1)
    with pytest.raises(ValueError):
        t.trim(a, 0)
    with pytest.raises(OutOfPages):
        t.extend(a, 7)          # more than max_pages
    b = t.open()
    with pytest.raises(OutOfPages):
        t.open()
    t.extend(a, 6)
    t.extend(b, 1)
    with pytest.raises(OutOfPages):
        t.extend(b, 2)
    assert t.lengths.tolist() == [6, 1]


@pytest.mark.parametrize("n,k,group", [(3, 1, 32), (5, 31, 32), (4, 200, 64), (2, 256, 256)])
def test_w4_layout_holds_the_codes(n, k, group):
    rng = np.random.default_rng(k)
    w = rng.standard_normal((n, k)).astype(np.float32)
    w[0] = 0
    q, s = K.w4_quantize(w, group)
    assert q.shape == (n, k) and s.shape == (n, -(-k // group)) and np.abs(q).max() <= 7 and (s[0] == 1).all()
    packed = K.w4_weight(q)
    assert packed.dtype == np.uint8 and packed.shape[1] % 16 == 0 and packed.shape[1] >= -(-k // 2)
    codes = np.stack([packed & 15, packed >> 4], -1).reshape(n, -1).astype(int) - 8
    assert np.array_equal(codes[:, :k], q) and (codes[:, k:] == 0).all()
    scale = np.repeat(s, group, 1)[:, :k]
    assert (np.abs(q * scale - w) <= scale * 0.5001).all()


# The rings between copying and computing warps (paged_attention.cuh): barriers known by the parity of a
# phase, tried in every order.

class _Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.phase = 0

    def arrive(self):
        assert self.pending > 0
        self.pending -= 1
        if self.pending == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def done(self, parity):
        return (self.phase - 1) & 1 == parity


def _ring_run(seed, feeders, warps, slots, steps):
    """Copies land in any order; returns what each computing warp read, in order."""
    rnd = random.Random(seed)
    full = {(w, i): _Barrier(2) for w in range(warps) for i in range(slots)}
    empty = {k: _Barrier(1) for k in full}
    data, read, flying = {}, [[] for _ in range(warps)], []
    fill, use = [[0, 0] for _ in range(warps)], [[0, 0] for _ in range(warps)]
    nxt_f, nxt_w = list(range(feeders)), list(range(warps))

    def forward(place):
        place[0] += 1
        if place[0] == slots:
            place[0], place[1] = 0, place[1] ^ 1

    for _ in range(200 * steps):
        if all(k >= steps for k in nxt_w):
            return read
        kind = rnd.randrange(3)
        if kind == 0:
            f = rnd.randrange(feeders)
            k = nxt_f[f]
            if k < steps:
                w = k % warps
                assert w % feeders == f
                at = (w, fill[w][0])
                if empty[at].done(fill[w][1] ^ 1):
                    data[at] = None
                    flying.append((at, k))
                    full[at].arrive()
                    forward(fill[w])
                    nxt_f[f] += feeders
        elif kind == 1 and flying:
            at, k = flying.pop(rnd.randrange(len(flying)))
            data[at] = k
            full[at].arrive()
        elif kind == 2:
            w = rnd.randrange(warps)
            if nxt_w[w] < steps:
                at = (w, use[w][0])
                if full[at].done(use[w][1]):
                    read[w].append(data[at])
                    empty[at].arrive()
                    forward(use[w])
                    nxt_w[w] += warps
    raise AssertionError("the ring stands still")


@pytest.mark.parametrize("feeders,warps", [(4, 12), (4, 8), (4, 4), (3, 6), (2, 6), (2, 4), (1, 3), (1, 2)])
@pytest.mark.parametrize("slots", [1, 2, 3, 4])
def test_every_warp_reads_its_own_steps_in_order(feeders, warps, slots):
    steps = 15 * warps + 1
    for seed in range(4):
        read = _ring_run(seed, feeders, warps, slots, steps)
        assert read == [list(range(w, steps, warps)) for w in range(warps)]
