"""The rows that sequences and groups of them have of a call (kmoe_paged_rows.h), compiled for the CPU: within the call's
rows whatever the arrays hold, and those of the members where they are ascending. No GPU needed."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CXX = shutil.which("g++") or shutil.which("c++")
pytestmark = pytest.mark.skipif(CXX is None, reason="no C++ compiler")

SOURCE = r"""
#include "kmoe_paged_rows.h"
extern "C" void rows(const int32_t *row_start, int a, int b, int64_t s_rows, int64_t *out) {
  const kmoe::RowRange first = kmoe::row_range(row_start[a], row_start[a + 1], s_rows);
  const kmoe::RowRange last = kmoe::row_range(row_start[b], row_start[b + 1], s_rows);
  const kmoe::RowRange all = kmoe::group_range(first, last);
  out[0] = first.r0, out[1] = first.n, out[2] = all.r0, out[3] = all.n;
}
"""


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    d = tmp_path_factory.mktemp("rows")
    (d / "rows.cpp").write_text(SOURCE)
    so = str(d / "rows.so")
    subprocess.run([CXX, "-std=c++17", "-O2", "-shared", "-fPIC", "-I", os.path.join(ROOT, "kestrel_amd", "csrc"), "-o", so,
                    str(d / "rows.cpp")], check=True)
    f = C.CDLL(so).rows
    f.restype, f.argtypes = None, [C.c_void_p, C.c_int, C.c_int, C.c_int64, C.c_void_p]

    def call(row_start, a, b, s_rows):
        """(r0, n) of sequence a, and of sequences a .. b together."""
        rs, out = np.ascontiguousarray(row_start, np.int32), np.zeros(4, np.int64)
        f(rs.ctypes.data, a, b, s_rows, out.ctypes.data)
        return tuple(out[:2].tolist()), tuple(out[2:].tolist())

    return call


def _all(rows, rs, s_rows):
    """Of every sequence and every group of neighbours: nothing outside the call's rows."""
    n = len(rs) - 1
    for a in range(n):
        for b in range(a, n):
            one, group = rows(rs, a, b, s_rows)
            for r0, k in (one, group):
                assert 0 <= r0 and 0 <= k and r0 + k <= s_rows, (rs, s_rows, a, b, one, group)
            yield a, b, one, group


@pytest.mark.parametrize("rs,s_rows", [([0, 1, 5, 7], 2), ([0, 1, 2 ** 31 - 2, 2 ** 31 - 1], 2), ([3, 3, 9, 9, 12], 9), ([0, 0, 0], 1), ([5, 7, 9], 4)])
def test_sequences_past_the_calls_rows(rows, rs, s_rows):
    """Ascending, as they have to be, but longer than the call: a group's rows are its members'."""
    for a, b, one, (r0, n) in _all(rows, rs, s_rows):
        assert one[1] == max(0, min(rs[a + 1], s_rows) - rs[a])
        assert list(range(r0, r0 + n)) == [r for r in range(s_rows) if rs[a] <= r < rs[b + 1]]


@pytest.mark.parametrize("seed", range(10))
def test_ascending_rows(rows, seed):
    rng = np.random.default_rng(seed)
    for _ in range(30):
        rs = np.sort(rng.integers(0, 40, rng.integers(2, 9)))
        s_rows = int(rng.integers(1, 45))
        for a, b, _, (r0, n) in _all(rows, rs, s_rows):
            assert list(range(r0, r0 + n)) == [r for r in range(s_rows) if rs[a] <= r < rs[b + 1]]


@pytest.mark.parametrize("seed", range(10))
def test_rows_that_make_no_sense_stay_inside(rows, seed):
    rng = np.random.default_rng(seed)
    assert list(_all(rows, [5, 2, 9, -4, 3, 100], 8))
    for _ in range(60):
        n = int(rng.integers(2, 8))
        rs = rng.choice([rng.integers(-10, 60, n), rng.integers(-2 ** 31, 2 ** 31, n)])
        assert list(_all(rows, rs, int(rng.choice([1, 8, 33, 1 << 22]))))
