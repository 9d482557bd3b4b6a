// kmoe_paged_rows.h — which rows of a call a sequence or a group of sequences has
// (internal; plain C++, so that its bounds are checked without a GPU).
#pragma once

#include <stdint.h>

namespace kmoe {

// Rows r0 .. r0 + n - 1, 0 <= r0 <= r0 + n <= the call's rows.
struct RowRange {
  int64_t r0, n;
};

// A sequence's rows lo .. hi - 1 as far as they are among the call's `rows`, whatever lo and hi
// are: a sequence past them has none and lies at their end.
constexpr RowRange row_range(int64_t lo, int64_t hi, int64_t rows) {
  lo = lo < 0 ? 0 : lo < rows ? lo : rows;
  hi = hi < rows ? hi : rows;
  return RowRange{lo, hi > lo ? hi - lo : 0};
}

// What begins with the rows of one sequence and ends with those of a later one.
constexpr RowRange group_range(RowRange first, RowRange last) {
  const int64_t end = last.r0 + last.n;
  return RowRange{first.r0, end > first.r0 ? end - first.r0 : 0};
}

}  // namespace kmoe
