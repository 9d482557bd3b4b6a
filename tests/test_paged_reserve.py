"""Positions for several sequences at once (kmoe_pages_append_many, PagedDecoder's reservation): all of them or none.
No GPU needed."""
import ctypes as C
import os

import numpy as np
import pytest

from kestrel_amd import kmoe
from tests.test_pages import BUDGET, INVALID, Model

pytestmark = pytest.mark.skipif(not os.path.exists(kmoe.LIB_PATH), reason="libkmoe.so not built (run __graft_entry__.build())")


def _decoder(n_pages, page, n_ctx=1000):
    """A PagedDecoder's account without a model; the copies that it asks for are listed."""
    from kestrel_amd.decoder import PagedDecoder

    dec = PagedDecoder.__new__(PagedDecoder)
    dec.account, dec.n_ctx, dec.window, dec.n_sink, dec.copied = kmoe.Pages(n_pages, page), n_ctx, 0, 0, []
    dec._copy = dec.copied.extend
    return dec


def test_a_reservation_that_fails_keeps_no_page():
    """A fork's first page of its own is not made for a call that another sequence's pages fail."""
    dec = _decoder(4, 32)
    dec._reserve({0: 40})
    dec.fork(0, 1)
    with pytest.raises(kmoe.KmoeError) as e:
        dec._reserve({0: 1, 2: 80})
    assert e.value.status == BUDGET
    assert dec.account.usage() == (2, 4) and not dec.copied and [dec.length(s) for s in range(3)] == [40, 40, 0]
    assert (dec.account.table([0], 2)[0] == dec.account.table([1], 2)[0]).all()
    dec._reserve({2: 64})  # the two pages that were free are
    assert dec.account.usage() == (4, 4)


class Many(Model):
    def append_many(self, want):
        before = {s: (self.p.table([s], 64)[0].tolist(), len(v)) for s, v in self.seqs.items()}
        used = self.p.usage()
        try:
            copies = self.p.append_many(want)
        except kmoe.KmoeError as e:
            assert e.status == BUDGET and self.p.usage() == used
            assert before == {s: (self.p.table([s], 64)[0].tolist(), self.p.length(s)) for s in self.seqs}
            for s in want:
                if s not in self.seqs:
                    with pytest.raises(kmoe.KmoeError):
                        self.p.length(s)
            return False
        assert len({d for _, d in copies}) == len(copies) and not {s for s, _ in copies} & {d for _, d in copies}
        for a, b in copies:  # in any order: no page is both copied from and onto
            for o in range(self.page):
                self.mem[b, o] = self.mem.get((a, o))
        for s, n in want.items():
            old = self.seqs.setdefault(s, [])
            at = len(old)
            old += list(range(self.next, self.next + n))
            self.next += n
            (row,), _ = self.p.table([s], 64)
            for i in range(at, len(old)):
                self.mem[int(row[i // self.page]), i % self.page] = old[i]
        return True


@pytest.mark.parametrize("seed", range(6))
def test_several_sequences_at_once(seed):
    """Sharers of a page that go on in one call each have a page of their own, the last keeps the shared one."""
    rng = np.random.default_rng(seed)
    m = Many(24, int(rng.choice([1, 4, 32])))
    done = [0, 0]
    for _ in range(300):
        some = list(m.seqs)
        op = rng.choice(["many", "many", "fork", "fork", "truncate", "drop"])
        if op == "many" or not some:
            pick = rng.permutation(10)[:int(rng.integers(1, 6))].tolist()
            done[m.append_many({s: int(rng.integers(0, 2 * m.page + 1)) for s in pick})] += 1
        else:
            s = int(rng.choice(some))
            n = int(rng.integers(0, len(m.seqs[s]) + 1))
            if op == "fork":
                free = [t for t in range(10) if t not in m.seqs]
                if free:
                    m.p.fork(s, free[0], n)
                    m.seqs[free[0]] = m.seqs[s][:n]
            elif op == "truncate":
                m.p.truncate(s, n)
                m.seqs[s] = m.seqs[s][:n]
            else:
                m.p.drop(s)
                del m.seqs[s]
        m.check()
    assert min(done) > 5, done


def test_refusals():
    p = kmoe.Pages(4, 32)
    p.append(1, 40)
    assert p.append_many({}) == [] and p.append_many({5: 0, 1: 0}) == [] and p.length(5) == 0
    for want in ({1: 3, 2: -1}, {2: 5, 1: 1 << 30}):
        with pytest.raises(kmoe.KmoeError) as e:
            p.append_many(want)
        assert e.value.status == INVALID and str(e.value)
    with pytest.raises(ValueError):
        p.append_many({1: 1, 2 ** 32 + 1: 1})
    ids, n, out = (C.c_uint32 * 2)(1, 1), (C.c_int64 * 2)(1, 1), (C.c_int32 * 2)()
    k = C.c_int32(7)
    for args in ((ids, n, 2, out, out, C.byref(k)), (ids, n, -1, out, out, C.byref(k)), (None, n, 1, out, out, C.byref(k)),
                 (ids, None, 1, out, out, C.byref(k)), (ids, n, 1, None, out, C.byref(k)), (ids, n, 1, out, None, C.byref(k)),
                 (ids, n, 1, out, out, None)):
        assert p.lib.kmoe_pages_append_many(p.h, *args) == INVALID
    assert p.lib.kmoe_pages_append_many(None, ids, n, 1, out, out, C.byref(k)) == INVALID
    assert p.length(1) == 40 and p.usage() == (2, 4)


def test_a_clone_goes_its_own_way():
    p = kmoe.Pages(6, 32)
    p.append(1, 40)
    p.fork(1, 2, 40)
    q = p.clone()
    assert q.append(1, 1) is not None and q.append(3, 96) is None and q.usage() == (6, 6)
    q.drop(2)
    assert p.usage() == (2, 6) and [p.length(s) for s in (1, 2)] == [40, 40]
    p.append(1, 1)
    p.drop(1)
    p.drop(2)
    assert p.usage() == (0, 6) and q.length(1) == 41 and q.usage()[0] == 5
    q.close()
    p.append(9, 6 * 32)
    assert p.lib.kmoe_pages_clone(None, C.byref(C.c_void_p())) == INVALID and p.lib.kmoe_pages_clone(p.h, None) == INVALID


@pytest.mark.parametrize("window,sink,had", [(40, 0, 0), (40, 5, 70), (1, 0, 33), (100, 40, 64)])
def test_a_window_serves_more_positions_than_pages(window, sink, had):
    """By steps where the pages are too few for all at once; every step's rows find what they see, and so does the
    sequence's old end until the call is over."""
    page = 32
    want = 12 * page
    steps = [{0: 16}] * (want // 16)
    need = -(-window // page) + 1 + -(-sink // page) + (-(-window // page) + 1 if had else 0) + 1
    dec = _decoder(need, page)
    dec.window, dec.n_sink = window, sink
    if had:
        dec._reserve({0: had})
        dec._trim([0])
    used = dec.account.usage()
    got, by_steps = dec._reserve({0: want}, steps)
    assert by_steps and got == {0: had or None} and dec.account.usage() == used
    n = had
    for step in steps:
        dec._append(step)
        (row,), _ = dec.account.table([0], 64)
        for pos in range(n, n + 16):
            for p in range(pos + 1):
                assert not (p > pos - window or p < sink) or row[p // page] >= 0
        n += 16
        dec._trim([0], got)
    if had:
        dec._back(got)
        (row,), _ = dec.account.table([0], 64)
        assert dec.length(0) == had and all(row[p // page] >= 0 for p in range(had) if p > had - window or p < sink)
    else:
        dec._back(got)
        assert dec.account.usage() == (0, need)


def test_a_window_that_does_not_fit_keeps_nothing():
    dec = _decoder(3, 32)
    dec.window = 100
    dec._reserve({0: 50})
    for steps in ([{0: 16}] * 20, [{0: 320}], []):
        with pytest.raises(kmoe.KmoeError) as e:
            dec._reserve({0: 320}, steps)
        assert e.value.status == BUDGET and dec.account.usage() == (2, 3) and dec.length(0) == 50
    dec.window = 0
    with pytest.raises(kmoe.KmoeError):
        dec._reserve({0: 320}, [{0: 16}] * 20)
    assert dec.account.usage() == (2, 3)


@pytest.mark.parametrize("status", [-3, -4])
def test_copies_that_fail_take_the_reservation_back(status):
    """Whatever the copies fail with, the positions are not kept, nor taken twice."""
    dec = _decoder(8, 32)
    dec.window = 100
    dec._reserve({0: 40})
    dec.fork(0, 1)

    def fails(pairs):
        assert pairs
        raise kmoe.KmoeError(status, "no")

    dec._copy = fails
    with pytest.raises(kmoe.KmoeError) as e:
        dec._reserve({0: 50, 2: 33}, [{0: 25, 2: 16}, {0: 25, 2: 17}])
    assert e.value.status == status and [dec.length(s) for s in range(3)] == [40, 40, 0]
