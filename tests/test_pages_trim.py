"""kmoe_pages_trim among the other calls: whatever is trimmed, truncated and forked, a sequence that is accepted holds
what its next row sees and can be written on. No GPU needed."""
import os

import numpy as np
import pytest

from kestrel_amd import kmoe
from tests.test_pages import INVALID, Model

pytestmark = pytest.mark.skipif(not os.path.exists(kmoe.LIB_PATH), reason="libkmoe.so not built (run __graft_entry__.build())")


def test_a_second_trim_of_the_front_keeps_what_the_first_gave_up():
    """The first positions are given up last: lengths whose pages went with the first trim stay refused."""
    p = kmoe.Pages(40, 32)
    p.append(1, 1000)
    assert p.trim(1, 100, 32) > 0
    with pytest.raises(kmoe.KmoeError) as e:
        p.truncate(1, 325)
    assert e.value.status == INVALID
    assert p.trim(1, 100, 0) == 1
    for f in (lambda: p.truncate(1, 325), lambda: p.fork(1, 2, 325)):
        with pytest.raises(kmoe.KmoeError) as e:
            f()
        assert e.value.status == INVALID
    assert p.length(1) == 1000 and p.append(1, 1) is None
    p.drop(1)
    assert p.usage() == (0, 40)


class Trimmed(Model):
    """Model that also knows the pages each sequence has given up, and the window of the last trim that gave any."""

    def __init__(self, n_pages, page):
        super().__init__(n_pages, page)
        self.gone, self.window = {}, {}

    def trim(self, s, window, sink):
        n, page = len(self.seqs[s]), self.page
        self.p.trim(s, window, sink)
        now = {i for i in range(n // page) if i * page >= sink and (i + 1) * page <= n - window + 1}
        if now - self.gone.setdefault(s, set()):
            self.window[s] = window
        self.gone[s] |= now

    def held(self, s, n):
        """Whether every position that a row at position n sees under the window is held, and n's own page."""
        if s not in self.window:
            return True
        lo = max(0, n - self.window[s] + 1)
        return all(i not in self.gone[s] for i in range(lo // self.page, -(-n // self.page)))

    def cut(self, call, s, n):
        """truncate or fork of s to n: whether it was accepted."""
        try:
            call()
        except kmoe.KmoeError as e:
            assert e.status == INVALID and n < len(self.seqs[s]) and not self.held(s, n)
            return False
        assert n == len(self.seqs[s]) or self.held(s, n)
        return True

    def check(self):
        super().check({(s, i) for s, g in self.gone.items() for i in g})


@pytest.mark.parametrize("seed", range(8))
def test_trims_between_truncations_and_forks(seed):
    rng = np.random.default_rng(seed)
    m = Trimmed(60, int(rng.choice([1, 4, 32])))
    for _ in range(500):
        op = rng.choice(["append", "append", "append", "fork", "truncate", "trim", "trim", "drop", "compact"])
        some = list(m.seqs)
        s = int(rng.choice(some)) if some else None
        if op == "append" or s is None:
            m.append(int(rng.integers(0, 8)), int(rng.integers(0, 5 * m.page)))
        elif op == "trim":
            m.trim(s, int(rng.integers(1, 4 * m.page + 1)), int(rng.choice([0, 0, 1, m.page, 2 * m.page + 1])))
        elif op == "drop":
            m.p.drop(s)
            for d in (m.seqs, m.gone, m.window):
                d.pop(s, None)
        elif op == "compact":
            src, dst = m.p.compact()
            for a, b in zip(src.tolist(), dst.tolist()):
                for o in range(m.page):
                    m.mem[b, o] = m.mem.pop((a, o), None)
        else:
            have = len(m.seqs[s])
            n = int(rng.integers(0, have + 1)) if rng.random() < 0.5 else max(0, have - int(rng.integers(0, m.page + 1)))
            if op == "truncate":
                if m.cut(lambda: m.p.truncate(s, n), s, n):
                    m.seqs[s] = m.seqs[s][:n]
                    m.gone[s] = {i for i in m.gone.get(s, ()) if i < -(-n // m.page)}
            else:
                t = int(rng.integers(8, 16))
                if t not in m.seqs and m.cut(lambda: m.p.fork(s, t, n), s, n):
                    m.seqs[t] = m.seqs[s][:n]
                    m.gone[t] = {i for i in m.gone.get(s, ()) if i < -(-n // m.page)}
                    if s in m.window:
                        m.window[t] = m.window[s]
        m.check()
    for s in list(m.seqs):
        m.p.drop(s)
    assert m.p.usage() == (0, 60)


@pytest.mark.parametrize("sink", [1 << 31, (1 << 63) - 1])
def test_first_positions_past_the_sequence(sink):
    """n_sink as large as it can be: every page is one of the first ones."""
    p = kmoe.Pages(40, 32)
    p.append(1, 1000)
    assert p.trim(1, 1, sink) == 0 and p.usage() == (32, 40)
    p.truncate(1, 5)


def test_back_to_the_first_positions():
    """Lengths inside the first pages that a trim leaves are what they are left for: forks and truncations go there."""
    p = kmoe.Pages(40, 32)
    p.append(1, 1000)
    p.trim(1, 100, 50)  # pages 0 and 1 stay, and 28 on
    for n in (65, 96, 500, 990 - 100 + 5):
        with pytest.raises(kmoe.KmoeError):
            p.fork(1, 2, n)
    for i, n in enumerate((0, 1, 32, 50, 64)):
        p.fork(1, 10 + i, n)
        assert p.length(10 + i) == n
    assert p.append(13, 1) is not None  # inside a shared page: a copy of its own
    used = p.usage()[0]
    p.truncate(1, 40)
    assert p.length(1) == 40 and p.usage()[0] == used - 4
    p.append(1, 200)
    (row,), _ = p.table([1], 8)
    assert (row >= 0).all()
    p.truncate(1, 0)


def test_a_sequence_ends_where_page_tables_do():
    """2^30 positions: the most that a page table of the kernels spans."""
    p = kmoe.Pages(4, 1 << 29)
    p.append(1, (1 << 30) - 1)
    with pytest.raises(kmoe.KmoeError) as e:
        p.append(1, 2)
    assert e.value.status == INVALID and p.length(1) == (1 << 30) - 1
    p.append(1, 1)
    with pytest.raises(kmoe.KmoeError) as e:
        p.append(1, 1)
    assert e.value.status == INVALID and p.usage() == (2, 4)


@pytest.mark.parametrize("seq", [2 ** 32 + 1, -(2 ** 32) + 1, -1, 2 ** 32])
def test_sequence_numbers_past_32_bits(seq):
    """Sequences are not named modulo 2^32."""
    p = kmoe.Pages(4, 32)
    p.append(1, 5)
    p.append(0, 3)
    p.append(2 ** 32 - 1, 2)
    for f in (lambda: p.append(seq, 1), lambda: p.drop(seq), lambda: p.truncate(seq, 1), lambda: p.fork(seq, 7, 1),
              lambda: p.fork(1, seq, 1), lambda: p.trim(seq, 1), lambda: p.length(seq), lambda: p.table([1, seq], 2),
              lambda: p.table(np.array([seq]), 2)):
        with pytest.raises(ValueError):
            f()
    assert [p.length(s) for s in (0, 1, 2 ** 32 - 1)] == [3, 5, 2] and p.usage() == (3, 4)
    assert p.table(np.array([1, 0]), 1)[1].tolist() == [5, 3]
