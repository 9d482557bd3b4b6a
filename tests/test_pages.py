"""kmoe_pages (the host's account of a paged cache) against a plain model that
holds every position's value by page: no GPU needed."""
import os

import numpy as np
import pytest

from kestrel_amd import kmoe

pytestmark = pytest.mark.skipif(not os.path.exists(kmoe.LIB_PATH), reason="libkmoe.so not built (run __graft_entry__.build())")

INVALID, BUDGET, NOT_LOADED = -1, -3, -5


class Model:
    """Cache contents as the calls' copies and stores leave them."""

    def __init__(self, n_pages, page):
        self.p, self.page, self.mem, self.seqs, self.next = kmoe.Pages(n_pages, page), page, {}, {}, 1

    def append(self, s, n):
        try:
            cp = self.p.append(s, n)
        except kmoe.KmoeError as e:
            assert e.status == BUDGET
            return False
        if cp:
            for o in range(self.page):
                self.mem[cp[1], o] = self.mem.get((cp[0], o))
        old = self.seqs.setdefault(s, [])
        at = len(old)
        old += list(range(self.next, self.next + n))
        self.next += n
        (row,), _ = self.p.table([s], 64)
        for i in range(at, len(old)):
            self.mem[int(row[i // self.page]), i % self.page] = old[i]
        return True

    def check(self, gone=()):
        held = set()
        for s, want in self.seqs.items():
            (row,), (n,) = self.p.table([s], 64)
            assert n == len(want) == self.p.length(s)
            cols = -(-n // self.page)
            assert (row[cols:] == -1).all()
            for i, x in enumerate(want):
                if (s, i // self.page) in gone:
                    continue
                assert self.mem[int(row[i // self.page]), i % self.page] == x
            held |= {int(x) for x in row[:cols] if x >= 0}
        assert self.p.usage()[0] == len(held)


@pytest.mark.parametrize("seed", range(6))
def test_any_order_of_calls_keeps_every_sequence(seed):
    rng = np.random.default_rng(seed)
    m = Model(40, int(rng.choice([1, 3, 32])))
    for _ in range(400):
        op = rng.choice(["append", "append", "append", "fork", "truncate", "drop", "compact"])
        some = list(m.seqs)
        s = int(rng.choice(some)) if some else None
        if op == "append" or s is None:
            m.append(int(rng.integers(0, 8)), int(rng.integers(0, 3 * m.page)))
        elif op == "fork":
            t, n = int(rng.integers(8, 16)), int(rng.integers(0, len(m.seqs[s]) + 1))
            if t in m.seqs:
                with pytest.raises(kmoe.KmoeError):
                    m.p.fork(s, t, n)
            else:
                m.p.fork(s, t, n)
                m.seqs[t] = m.seqs[s][:n]
        elif op == "truncate":
            n = int(rng.integers(0, len(m.seqs[s]) + 1))
            m.p.truncate(s, n)
            m.seqs[s] = m.seqs[s][:n]
        elif op == "drop":
            m.p.drop(s)
            del m.seqs[s]
        else:
            cap = None if rng.random() < 0.5 else int(rng.integers(0, 4))
            src, dst = m.p.compact(cap)
            assert not set(src) & set(dst) and len(set(dst)) == len(dst)
            for a, b in zip(src.tolist(), dst.tolist()):
                for o in range(m.page):
                    m.mem[b, o] = m.mem.pop((a, o), None)
            if cap is None:
                used = m.p.usage()[0]
                assert all(x < used for t in m.seqs for x in m.p.table([t], 64)[0][0])
        m.check()
    for s in list(m.seqs):
        m.p.drop(s)
    assert m.p.usage() == (0, 40)


def test_append_past_the_pool_changes_nothing():
    p = kmoe.Pages(4, 32)
    assert p.append(1, 70) is None and p.usage() == (3, 4)
    with pytest.raises(kmoe.KmoeError) as e:
        p.append(1, 27 + 32)
    assert e.value.status == BUDGET and p.length(1) == 70 and p.usage() == (3, 4)
    with pytest.raises(kmoe.KmoeError):
        p.append(2, 33)
    with pytest.raises(kmoe.KmoeError) as e:
        p.length(2)
    assert e.value.status == NOT_LOADED
    p.fork(1, 3, 70)
    p.append(1, 0)  # nothing new: nothing to copy
    assert p.append(1, 26) is not None and p.usage() == (4, 4)  # its own copy of the shared page
    with pytest.raises(kmoe.KmoeError) as e:
        p.append(1, 1)
    assert e.value.status == BUDGET and p.length(1) == 96
    assert p.append(3, 1) is None and p.append(3, 25) is None  # the page is its own now


def test_fork_at_a_page_border_copies_nothing():
    p = kmoe.Pages(8, 32)
    p.append(0, 64)
    p.fork(0, 1, 64)
    assert p.append(0, 1) is None and p.append(1, 1) is None and p.usage() == (4, 8)
    p.fork(0, 2, 0)  # of no positions: holds nothing
    assert p.length(2) == 0 and p.usage() == (4, 8)


@pytest.mark.parametrize("window,sink,n", [(1, 0, 64), (1, 0, 65), (10, 0, 200), (33, 4, 200), (64, 33, 257), (300, 4, 200)])
def test_trim_keeps_what_later_rows_see(window, sink, n):
    page = 32
    p = kmoe.Pages(40, page)
    p.append(5, n)
    freed = p.trim(5, window, sink)
    (row,), _ = p.table([5], 40)
    for pos in range(n):  # the next row, at position n, and every later one
        seen = pos > n - window or pos < sink
        assert not seen or row[pos // page] >= 0
    cols = -(-n // page)
    want = [i for i in range(cols) if i * page >= sink and (i + 1) * page <= n - window + 1]
    assert freed == len(want) == (row[:cols] == -1).sum() and p.usage()[0] == cols - freed
    assert p.trim(5, window, sink) == 0
    if freed:
        with pytest.raises(kmoe.KmoeError) as e:
            p.truncate(5, (want[-1] + 1) * page - 1)
        assert e.value.status == INVALID
        with pytest.raises(kmoe.KmoeError):
            p.fork(5, 6, (want[-1] + 1) * page - 1)
    p.fork(5, 7, n)
    p.append(7, 1)
    p.drop(5)
    p.drop(7)
    assert p.usage()[0] == 0


def test_refusals():
    for n, page in ((0, 32), (-1, 32), (4, 0), (1 << 31, 32)):
        with pytest.raises(kmoe.KmoeError):
            kmoe.Pages(n, page)
    p = kmoe.Pages(4, 32)
    p.append(1, 40)
    for f, st in ((lambda: p.append(1, -1), INVALID), (lambda: p.append(1, (1 << 31) - 1), INVALID),
                  (lambda: p.fork(9, 2, 0), NOT_LOADED), (lambda: p.fork(1, 1, 0), INVALID),
                  (lambda: p.fork(1, 2, 41), INVALID), (lambda: p.fork(1, 2, -1), INVALID),
                  (lambda: p.truncate(1, 41), INVALID), (lambda: p.truncate(9, 0), NOT_LOADED),
                  (lambda: p.drop(9), NOT_LOADED), (lambda: p.trim(1, 0), INVALID), (lambda: p.trim(1, 5, -1), INVALID),
                  (lambda: p.table([1], 1), INVALID), (lambda: p.table([1, 9], 8), NOT_LOADED),
                  (lambda: p.compact(-1), INVALID)):
        with pytest.raises(kmoe.KmoeError) as e:
            f()
        assert e.value.status == st and str(e.value)
    assert p.length(1) == 40 and p.usage() == (2, 4)


def test_page_bytes():
    import ctypes as C

    lib, n = kmoe.load_library(), C.c_uint64()
    for t, per in ((kmoe.F16, 2 * 64 * 4), (kmoe.Q8_0, 2 * 64 * 34 // 16)):
        for hd in (64, 128):
            d = kmoe.PagedDesc(t, 3, hd, 64, 1)
            assert lib.kmoe_paged_page_bytes(C.byref(d), C.byref(n)) == 0
            assert n.value == kmoe.PagedKV(t, 3, hd, 64).page_bytes == 3 * hd * per // 2
    for bad in ((0, 3, 64, 64), (1, 0, 64, 64), (1, 3, 96, 64), (1, 3, 64, 48)):
        assert lib.kmoe_paged_page_bytes(C.byref(kmoe.PagedDesc(*bad, 1)), C.byref(n)) == INVALID
