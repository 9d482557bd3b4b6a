"""The positions that a row's plain form goes through (kmoe_paged_walk.h), compiled for the CPU: every visible position
that has a page, once, and steps that the table bounds, not the length. No GPU needed."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CXX = shutil.which("g++") or shutil.which("c++")
pytestmark = pytest.mark.skipif(CXX is None, reason="no C++ compiler")
LOOK = 1024  # columns that a work-group's search takes at a time

SOURCE = r"""
#include "kmoe_paged_walk.h"
extern "C" int64_t walk(int64_t pos, int64_t lo, int64_t sink, int64_t cols, int page, const int8_t *has, int look,
                        int64_t *finds, uint16_t *seen) {
  int64_t blocks = 0;
  *finds = 0;
  auto page_of = [&](int64_t col) { return col < cols && (!has || has[col]); };
  kmoe::plain_walk(pos, lo, sink, cols * page, page,
    [&](int64_t p0) {
      ++blocks;
      bool some = false;
      for (int64_t p = p0; p < p0 + 256; ++p)
        if (p <= pos && (p >= lo || p < sink) && page_of(p / page)) {
          some = true;
          if (seen) ++seen[p];
        }
      return some;
    },
    [&](int64_t col) {
      ++*finds;
      int n = 0;
      while (n < look && !page_of(col + n)) ++n;
      return n;
    });
  return blocks;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cpp").write_text(SOURCE)
    so = str(d / "walk.so")
    subprocess.run([CXX, "-std=c++17", "-O2", "-shared", "-fPIC", "-I", os.path.join(ROOT, "kestrel_amd", "csrc"), "-o", so,
                    str(d / "walk.cpp")], check=True)
    f = C.CDLL(so).walk
    f.restype, f.argtypes = C.c_int64, [C.c_int64] * 4 + [C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]

    def call(pos, window, sink, cols, page, has=None, seen=None):
        n = C.c_int64()
        lo = pos - window + 1 if 0 < window <= pos else 0
        p = [x.ctypes.data if x is not None else None for x in (has, seen)]
        blocks = f(pos, lo, sink, cols, page, p[0], LOOK, C.byref(n), p[1])
        return blocks, n.value

    return call


@pytest.mark.parametrize("seed", range(10))
def test_every_visible_position_with_a_page_once(walk, seed):
    rng = np.random.default_rng(seed)
    for _ in range(60):
        page = int(rng.choice([32, 64, 128, 256]))
        cols = int(rng.integers(0, 60))
        has = (rng.random(max(cols, 1)) < rng.choice([0.0, 0.05, 0.5, 1.0])).astype(np.int8)
        pos = int(rng.choice([rng.integers(-3, cols * page + 600), 2 ** 31 - 2]))
        window = int(rng.choice([0, 1, 255, 256, 257, rng.integers(1, 9000), max(1, pos - int(rng.integers(0, 9000)))]))
        sink = int(rng.choice([0, 1, 5, 256, 700, 2 ** 30])) if window else 0
        seen = np.zeros(cols * page + 256, np.uint16)
        blocks, finds = walk(pos, window, sink, cols, page, has, seen)
        p = np.arange(len(seen))
        want = (p <= pos) & ((p > pos - window if window else p >= 0) | (p < sink)) & (p < cols * page)
        want &= has[np.minimum(p // page, max(cols, 1) - 1)] > 0
        assert np.array_equal(seen, want.astype(np.uint16))
        assert blocks <= cols * page // 256 + 1 and finds <= blocks


@pytest.mark.parametrize("page", [32, 256])
@pytest.mark.parametrize("window,sink", [(0, 0), (1, 0), (2 ** 31 - 1, 0), (2 ** 30, 7), (100, 2 ** 30)])
def test_a_length_past_the_table_costs_no_more_than_the_table(walk, page, window, sink):
    for cols in (0, 1, 5):
        blocks, _ = walk(2 ** 31 - 2, window, sink, cols, page)
        assert blocks <= -(-cols * page // 256)


def test_missing_pages_are_passed_over_together(walk):
    cols = 1 << 20
    has = np.zeros(cols, np.int8)
    has[777777] = 1
    seen = np.zeros(cols * 32 + 256, np.uint16)
    blocks, finds = walk(2 ** 31 - 2, 0, 0, cols, 32, has, seen)
    assert seen.sum() == 32 and seen[777777 * 32] == 1
    assert finds <= cols // LOOK + 2 and blocks <= finds + 2
