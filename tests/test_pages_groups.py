"""kmoe_pages_groups: which sequences of a batch share pages (host only, no GPU),
against all partitions of small batches and plain page tables."""
import ctypes as C
import os

import numpy as np
import pytest

from kestrel_amd import kmoe

pytestmark = pytest.mark.skipif(not os.path.exists(kmoe.LIB_PATH), reason="libkmoe.so not built")
PAGE = 4


def _saved(p, seqs, groups):
    """Pages that are not read again, and that every group's members hold the same ones."""
    order, start, shared = groups
    assert sorted(order.tolist()) == list(range(len(seqs))) and start[0] == 0 and (np.diff(start) >= 2).all()
    assert (order[start[-1]:] == np.sort(order[start[-1]:])).all()
    if not len(seqs):
        return 0
    t, _ = p.table(seqs, max(1, max(-(-p.length(s) // PAGE) for s in seqs)))
    n = 0
    for i, k in enumerate(shared):
        m = t[order[start[i]:start[i + 1]], :k]
        assert k > 0 and (m == m[0]).all() and (m >= 0).all()
        n += (start[i + 1] - start[i] - 1) * int(k)
    return n


def _tree(seed, n):
    """n sequences of random forks, some of whose pages are trimmed."""
    rng = np.random.default_rng(seed)
    p = kmoe.Pages(4000, PAGE)
    p.append(0, int(rng.integers(1, 30)))
    for s in range(1, n):
        src = int(rng.integers(0, s))
        if rng.random() < 0.2:
            p.append(s, int(rng.integers(1, 20)))
        else:
            try:
                p.fork(src, s, int(rng.integers(0, p.length(src) + 1)))
            except kmoe.KmoeError:  # its window was trimmed there
                p.fork(src, s, p.length(src))
            if rng.random() < 0.8:
                p.append(s, int(rng.integers(1, 20)))
        if rng.random() < 0.1:
            p.trim(s, 6, 2)
    return p


def _best(p, seqs):
    """The most pages that any partition of the sequences saves."""
    t, _ = p.table(seqs, 40)

    def common(m):
        same = ((t[m] == t[m[0]]) & (t[m] >= 0)).all(0)
        return int(np.argmin(same)) if not same.all() else t.shape[1]

    def go(rest):
        if not rest:
            return 0
        best = 0
        for mask in range(1 << (len(rest) - 1)):
            with_ = [rest[0]] + [x for i, x in enumerate(rest[1:]) if mask >> i & 1]
            best = max(best, (len(with_) - 1) * common(with_) + go([x for x in rest if x not in with_]))
        return best

    return go(list(range(len(seqs))))


@pytest.mark.parametrize("seed", range(40))
def test_no_partition_saves_more(seed):
    """Up to seven sequences: as many pages as the best of all partitions."""
    n = 2 + seed % 6
    p = _tree(seed, n)
    seqs = np.random.default_rng(seed).permutation(n).tolist()
    assert _saved(p, seqs, p.groups(seqs)) == _best(p, seqs)


@pytest.mark.parametrize("n", [1, 64, 300])
def test_large_batches(n):
    p = _tree(n, n)
    got = p.groups(range(n))
    assert (_saved(p, list(range(n)), got) > 0) == (n > 1)


def test_one_prompt_and_its_forks():
    p = kmoe.Pages(100, PAGE)
    p.append(5, 18)
    for s in range(4):
        p.fork(5, 10 + s, 18)
    p.append(3, 9)
    p.append_many({s: 1 for s in (10, 11, 12, 13, 3)})
    order, start, shared = p.groups([10, 3, 13, 11, 12])
    assert start.tolist() == [0, 4] and shared.tolist() == [4] and sorted(order[:4].tolist()) == [0, 2, 3, 4] and order[4] == 1
    # 3 members read 4 pages of 4 positions again
    for least, groups in ((48, 1), (49, 0), (10 ** 12, 0), (0, 1)):
        assert len(p.groups([10, 3, 13, 11, 12], least)[2]) == groups
    assert len(p.groups([10, 3])[2]) == 0 and len(p.groups([])[2]) == 0


def test_a_chain_of_forks_is_no_recursion():
    """Each of 4096 sequences goes on from the one before by a page: runs nest as deep as there are sequences."""
    p = kmoe.Pages(5000, 1)
    p.append(0, 1)
    for s in range(1, 4096):
        p.fork(s - 1, s, s)
        p.append(s, 1)
    order, start, shared = p.groups(range(4096))
    assert start[-1] > 0 and shared.max() > 0


def test_refusals():
    p = kmoe.Pages(10, PAGE)
    p.append(1, 5)
    p.append(2, 5)
    for seqs in ([1, 3], [1, 2, 1]):
        with pytest.raises(kmoe.KmoeError):
            p.groups(seqs)
    with pytest.raises(kmoe.KmoeError):
        p.groups([1, 2], -1)
    with pytest.raises(ValueError):
        p.groups([-1])
    n, x = C.c_int32(), np.zeros(4, np.int32)
    f = p.lib.kmoe_pages_groups
    ids = np.array([1, 2], np.uint32)
    ok = [p.h, ids.ctypes.data, 2, 1, x.ctypes.data, np.zeros(4, np.int32).ctypes.data, x.ctypes.data, C.byref(n)]
    for i in (0, 1, 4, 5, 6, 7):
        bad = list(ok)
        bad[i] = None
        assert f(*bad) == -1
    assert f(p.h, None, -1, 1, None, x.ctypes.data, None, C.byref(n)) == -1


def test_as_many_sequences_as_a_batch_takes():
    p = kmoe.Pages(10, PAGE)
    p.append(0, 2 * PAGE)
    for i in range(1, 4097):
        p.fork(0, i, 2 * PAGE)
    order, start, shared = p.groups(range(4096))
    assert start.tolist() == [0, 4096] and shared.tolist() == [2] and sorted(order.tolist()) == list(range(4096))
    with pytest.raises(kmoe.KmoeError, match="at most 4096"):
        p.groups(range(4097))
