// kmoe_scan.h — sums along a wave's lanes by lane moves (internal): within rows of 16
// lanes, then row 0's and 2's last lanes onto rows 1 and 3, then lane 31 onto the upper
// half. Six steps of two to four instructions; through LDS a step takes a round trip.
#pragma once

#include "kmoe_device.h"

namespace kmoe {

// x of the lane that CTRL names; lanes without one, and rows that are not in ROWS, get `none`.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t none, uint64_t x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)none, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)(none >> 32), (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xf, false);
  return (uint64_t)hi << 32 | lo;
}
// row_shr 1, 2, 4, 8, row_bcast 15 and 31, and the rows that take each.
#define KMOE_ALONG_LANES(STEP) \
  STEP(0x111, 0xf) STEP(0x112, 0xf) STEP(0x114, 0xf) STEP(0x118, 0xf) STEP(0x142, 0xa) STEP(0x143, 0xc)

// Inclusive sums; lane 63 has the whole.
__device__ __forceinline__ uint64_t wave_scan(uint64_t x) {
#define KMOE_STEP(CTRL, ROWS) x += dpp_u64<CTRL, ROWS>(0, x);
  KMOE_ALONG_LANES(KMOE_STEP)
#undef KMOE_STEP
  return x;
}
__device__ __forceinline__ int wave_scan_i(int x) {
#define KMOE_STEP(CTRL, ROWS) x += __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
  KMOE_ALONG_LANES(KMOE_STEP)
#undef KMOE_STEP
  return x;
}
// The least and the largest so far; lane 63 has the whole's.
__device__ __forceinline__ void wave_range(uint64_t &mn, uint64_t &mx) {
#define KMOE_STEP(CTRL, ROWS)                        \
  {                                                  \
    const uint64_t a = dpp_u64<CTRL, ROWS>(mn, mn);  \
    const uint64_t b = dpp_u64<CTRL, ROWS>(mx, mx);  \
    mn = a < mn ? a : mn;                            \
    mx = b > mx ? b : mx;                            \
  }
  KMOE_ALONG_LANES(KMOE_STEP)
#undef KMOE_STEP
}
// Sum over aligned groups of W lanes (8 or 16), to all of them.
template <int W>
__device__ __forceinline__ double group_sum_d(double x) {
#define KMOE_STEP(CTRL) x += __builtin_bit_cast(double, dpp_u64<CTRL, 0xf>(0, __builtin_bit_cast(uint64_t, x)));
  KMOE_STEP(kDppXor1)
  KMOE_STEP(kDppXor2)
  KMOE_STEP(kDppHalfMirror)
  if constexpr (W == 16) KMOE_STEP(kDppMirror)
#undef KMOE_STEP
  return x;
}

}  // namespace kmoe
