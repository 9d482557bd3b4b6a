"""kmoe_pages_groups where a group has to save something: sequences whose nearest common beginning saves too little by
itself still share a shorter one (host only, no GPU)."""
import os

import numpy as np
import pytest

from kestrel_amd import kmoe
from tests.test_pages_groups import PAGE, _saved, _tree

pytestmark = pytest.mark.skipif(not os.path.exists(kmoe.LIB_PATH), reason="libkmoe.so not built")


def _best(p, seqs, least):
    """The most pages that any partition saves whose groups save `least` positions each."""
    t, _ = p.table(seqs, 40)

    def common(m):
        same = ((t[m] == t[m[0]]) & (t[m] >= 0)).all(0)
        return int(np.argmin(same)) if not same.all() else t.shape[1]

    def go(rest):
        best = 0
        for mask in range(1 << (len(rest) - 1)) if rest else ():
            m = [rest[0]] + [x for i, x in enumerate(rest[1:]) if mask >> i & 1]
            n = (len(m) - 1) * common(m)
            if len(m) == 1 or n * PAGE >= least:
                best = max(best, n + go([x for x in rest if x not in m]))
        return best

    return go(list(range(len(seqs))))


@pytest.mark.parametrize("seed", range(40))
def test_no_partition_of_groups_that_save_enough_saves_more(seed):
    n = 2 + seed % 6
    p = _tree(seed, n)
    seqs = np.random.default_rng(seed).permutation(n).tolist()
    for least in (0, 1, 3 * PAGE, 8 * PAGE + 1, 20 * PAGE):
        order, start, shared = got = p.groups(seqs, least)
        assert all((start[i + 1] - start[i] - 1) * int(k) * PAGE >= least for i, k in enumerate(shared))
        assert _saved(p, seqs, got) == _best(p, seqs, least)


def test_two_continuations_of_each_of_many_forks():
    """16 forks of a beginning of 20 pages, each with 21 pages of its own, then forked: a pair saves 41 pages, more
    together than the 31 * 20 of all by their beginning, which they are grouped by where a pair is not enough."""
    p = kmoe.Pages(4000, PAGE)
    p.append(0, 20 * PAGE)
    for i in range(16):
        p.fork(0, 10 + i, 20 * PAGE)
        p.append(10 + i, 21 * PAGE)
        p.fork(10 + i, 100 + i, 41 * PAGE)
        p.append_many({10 + i: 1, 100 + i: 1})
    seqs = [*range(10, 26), *range(100, 116)]
    for least, groups, saved in ((41 * PAGE, 16, 16 * 41), (41 * PAGE + 1, 1, 31 * 20), (31 * 20 * PAGE, 1, 31 * 20), (31 * 20 * PAGE + 1, 0, 0)):
        got = p.groups(seqs, least)
        assert len(got[2]) == groups and _saved(p, seqs, got) == saved
