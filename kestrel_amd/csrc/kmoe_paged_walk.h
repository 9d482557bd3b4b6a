// kmoe_paged_walk.h — the positions that a row's plain form goes through
// (internal; plain C++, so that its bounds are checked without a GPU).
#pragma once

#include <stdint.h>

namespace kmoe {

// Blocks of 256 positions in which the row at position `pos` of a sequence may see
// something (positions lo .. pos, and those below `sink`), within a table of `cap`
// positions on pages of `page` (a divisor of 256): the sequence's length is the
// caller's and may be past its pages by any amount. block(p0) works the block at p0
// and says whether any of its visible positions has a page; where none has,
// find(col) says how many columns of the table from col on name no page (as far as
// it looked, a multiple of 8 and at least 8 where it found none), and they are passed over.
template <class Block, class Find>
constexpr void plain_walk(int64_t pos, int64_t lo, int64_t sink, int64_t cap, int page, Block &&block, Find &&find) {
  const int64_t end = pos < cap ? pos + 1 : cap;
  for (int64_t p0 = 0;;) {
    if (p0 >= sink && p0 + 256 <= lo) p0 = lo / 256 * 256;  // between the first positions and the window
    if (p0 >= end) return;
    const bool some = block(p0);
    p0 += 256;
    if (!some && p0 < end) p0 += (int64_t)find(p0 / page) * page / 256 * 256;
  }
}

}  // namespace kmoe
