// kmoe_sample.hip — the next token of every row of logits: temperature, top-k,
// top-p, min-p, and a draw by a given random number.
//
// A row's weights are w_i = exp((l_i - max l) / T). Kept are, in the order of
// descending l (equal ones by index), the first top_k, of those the shortest
// beginning that holds top_p of their weight, of those the ones with w_i >= min_p:
// always a beginning of that order, given by its last value and how many equal to
// it are in. The token drawn is the first kept one, by index, at which the running
// sum passes u times the sum.
//
// Which token that is depends on borders between sums of many thousand weights, so
// an exponential in 32 bits would move about one draw in a hundred. Weights are
// 64-bit floats, off by 2^-52, and summed as whole multiples of 2^-43: sums of
// whole numbers do not depend on their order, so neither atomics nor the way a row
// is shared out change a result. 2^20 weights of at most 1 fit 63 bits; what is
// rounded off is 2^-44 of the largest weight each, at most 2^-24 of the sum (the
// step of u) in all. The sum of a whole long row, which the draw without a cut and top_p
// go by, is that of its chunks, each summed by its own largest logit before the row's is
// known: rounded otherwise than the row's weights, but the same on every path of a row.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "kmoe_device.h"
#include "kmoe_launch.h"
#include "kmoe_scan.h"

namespace kmoe {
namespace {

typedef unsigned long long u64;
// Threads of a work-group: with 1024, every step between two barriers is issued four
// times per SIMD, and most steps of a row are short (256 rows without a cut: 12 us, with 256 7).
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kFix = 43;    // weights in units of 2^-43
constexpr int kBins = 1024, kBinsEach = kBins / kThreads;
constexpr int kTab = 256;
constexpr int kGroup = 64, kChunk = 1024;  // elements of which k_sample_stats finds the largest, and the sum
constexpr int kCand = 4096, kGroups = 1024, kFewGroups = 256;
constexpr int kFew = 1024;  // elements of a bin that are compared one with another
constexpr int kParts = 16;  // work-groups that share a row at most
constexpr int kSegment = 1024;  // elements of which a draw knows the sum
// Distances from the largest logit that the even bins tell apart: to the lowest that is binned,
// at most this (a mask's -10^9 is none of the others' business) and 24 T, where
// weights are what counts 24 T.
constexpr float kSpan = 64.0f, kSpanT = 24.0f;

// The larger of two that are no signalling NaNs (fmaxf quiets its operands first).
__device__ __forceinline__ float max2(float a, float b) {
  asm("v_max_f32 %0, %1, %2" : "=v"(a) : "v"(a), "v"(b));
  return a;
}
// NaN as -inf. Order of the logits as whole numbers: the larger the logit, the smaller
// its rank (-0 as 0).
__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return ~(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u));
}
__device__ __forceinline__ float of_rank(uint32_t r) {
  const uint32_t k = ~r;
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// What one row is drawn by.
struct Row {
  double max;    // largest logit
  double inv_t;  // 256 / (T log 2)
  float top, scale;  // largest logit; bins per unit of logit
  double min_w;  // min_p in units
  float u;
};

// Elements of a row: of the logits themselves, or candidates in LDS, in the order of their index.
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));
struct Logits {
  const float *l;
  int n;
  __device__ __forceinline__ float at(int i) const { return clean(l[i]); }
};
struct Candidates {
  const float *l;
  int n;
  __device__ __forceinline__ float at(int i) const { return l[i]; }
};

// 2^(i / 256)
__device__ __forceinline__ void make_table(double *tab) {
  static_assert(kTab == kThreads, "one entry a thread");
  tab[threadIdx.x] = exp2((double)threadIdx.x / kTab);
}

// A weight in units: z = 256 log2 of it is i + f, |f| <= 1/2, and 2^(z / 256) a power of two
// times 2^((i mod 256) / 256) (LDS) times the exponential of f log(2) / 256 by its
// series, whose fifth power's term is 2^-54.5. i comes out of z's sum with 1.5 2^52,
// whose last bit is 1. The largest logit's weight is 2^43 exactly. Below 2^-44 (-31
// nats: z = -11450) the weight rounds to no unit, whatever it is. A NaN is an infinite
// largest logit's distance from itself.
// MAY_BE_INF: the largest logit may be infinite.
template <bool MAY_BE_INF = true>
__device__ __forceinline__ double weight(const Row &r, float l, const double *tab) {
  double z = ((double)l - r.max) * r.inv_t;
  if constexpr (MAY_BE_INF) z = fmin(z, 0.0);
  z = fmax(z, -11450.0);
  const double s = z + 0x1.8p52;
  const int i = (int)(uint32_t)__double_as_longlong(s);
  const double f = z - (s - 0x1.8p52);
  double y = fma(f, 0x1.3b2ab6fba4e77p-39, 0x1.c6b08d704a0c0p-29);  // (log(2) / 256)^k / k!
  y = fma(f, y, 0x1.ebfbdff82c58fp-19);
  y = fma(f, y, 0x1.62e42fefa39efp-9);
  y = f * y;
  const double t = tab[i & (kTab - 1)];
  const double u = __hiloint2double(__double2hiint(t) + (((i >> 8) + kFix) << 20), __double2loint(t));
  return fma(u, y, u);
}
// To the nearest unit: 2^52 and a number below it have a last bit of 1.
__device__ __forceinline__ u64 fixed(double w) { return (u64)__double_as_longlong(w + 0x1p52) & ((1ull << 52) - 1); }

// Even bins by the distance from the largest logit (not descending where the logits
// descend); an infinite largest one's own distance is a NaN: bin 0.
__device__ __forceinline__ int bin_of(const Row &r, float l) {
  return (int)__builtin_amdgcn_fmed3f((r.top - l) * r.scale, 0.0f, (float)(kBins - 1));
}

struct Shared {
  double tab[kTab];
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 red[kWaves];
  uint32_t redi[kWaves];
  float redf[2][kWaves];
  u64 part[kParts];
  u64 before, above, ties;
  int at, n;
  // elements of one bin
  uint32_t rank[64];
  u64 w[64];
  // candidates, and the groups that they are in with how many candidates each has
  float cand[kCand];
  int index[kCand];
  uint16_t group[kGroups], in_group[128];
};

// Exclusive scan over the work-group's threads, and the total.
__device__ __forceinline__ u64 block_scan(u64 x, u64 &total, Shared &sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 in = wave_scan(x);
  lds_barrier();  // (the last call's sums are read)
  if (lane == 63) sh.red[wave] = in;
  lds_barrier();
  u64 before = in - x;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const u64 y = sh.red[w];
    if (w < wave) before += y;
    total += y;
  }
  return before;
}

// The first of EACH * kThreads bins at which the running sum of hist reaches `target` (1 .. the
// total), and the sum before it.
template <int EACH, class T>
__device__ __forceinline__ int crossing(const T *hist, u64 target, u64 &before, Shared &sh) {
  const int t = threadIdx.x;
  u64 x[EACH], s = 0, total;
#pragma unroll
  for (int e = 0; e < EACH; ++e) s += x[e] = hist[EACH * t + e];
  u64 y = block_scan(s, total, sh);
  if (y < target && y + s >= target) {
    int e = 0;
#pragma unroll
    for (int k = 0; k < EACH - 1; ++k)
      if (e == k && y + x[k] < target) {
        y += x[k];
        ++e;
      }
    sh.at = EACH * t + e;
    sh.before = y;
  }
  lds_barrier();
  before = sh.before;
  return sh.at;
}
template <class T>
__device__ __forceinline__ int crossing(const T *hist, u64 target, u64 &before, Shared &sh) {
  return crossing<kBinsEach>(hist, target, before, sh);
}
// The sum of all bins below `end`.
template <class T>
__device__ __forceinline__ u64 sum_below(const T *hist, int end, Shared &sh) {
  const int t = threadIdx.x;
  u64 s = 0, total;
#pragma unroll
  for (int e = 0; e < kBinsEach; ++e) s += kBinsEach * t + e < end ? hist[kBinsEach * t + e] : 0;
  block_scan(s, total, sh);
  return total;
}

// f(i, l) for every element i, a work-group together; loads of a row wait for each other
// as little as the registers allow (32 elements a thread: a flat row's bin 15 -> 7 us).
template <class F>
__device__ __forceinline__ void each(const Candidates &src, F &&f) {
  for (int i = threadIdx.x; i < src.n; i += kThreads) f(i, src.at(i));
}
template <class F>
__device__ __forceinline__ void each(const Logits &src, F &&f) {
  constexpr int U = 8;
  const int n4 = src.n & ~3;
  for (int i0 = 4 * threadIdx.x; i0 < n4; i0 += 4 * U * kThreads) {
    f32x4a4 x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + 4 * j * kThreads;
      x[j] = *(const f32x4a4 *)(src.l + (i < n4 ? i : i0));
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + 4 * j * kThreads;
      if (i >= n4) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) f(i + e, clean(x[j][e]));
    }
  }
  if ((int)threadIdx.x < src.n - n4) f(n4 + threadIdx.x, src.at(n4 + threadIdx.x));
}

template <class T>
__device__ __forceinline__ void clear(T *h) {
#pragma unroll
  for (int e = 0; e < kBinsEach; ++e) h[kThreads * e + threadIdx.x] = 0;
}

// Sum of f(i, l) over the elements, to every thread.
template <class S, class F>
__device__ __forceinline__ u64 sum_of(const S &src, Shared &sh, F &&f) {
  u64 s = 0, total;
  each(src, [&](int i, float l) { s += f(i, l); });
  block_scan(s, total, sh);
  return total;
}

// A beginning of the order: values above v, and the first `ties` of those equal to it.
struct Cut {
  float v;
  u64 ties;
};

// Where the running sum over the elements of an even bin whose rank is below `limit`
// reaches target (1 .. their sum): the value, what is left of the target there, and
// (above) the weight of the bin's elements before it. MASS: sums of weights, otherwise
// numbers of elements. Digit by digit of the rank; the even bins' sums of that kind are
// used up.
template <bool MASS, class S>
__device__ __forceinline__ Cut cut_by_digits(const Row &r, const S &src, int bin, uint32_t limit, u64 target, u64 &above,
                                             Shared &sh) {
  uint32_t found = 0;
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    lds_barrier();
    if (MASS) sh.mass[threadIdx.x] = 0;
    else sh.count[threadIdx.x] = 0;
    lds_barrier();
    each(src, [&](int, float l) {
      if (bin_of(r, l) != bin) return;
      const uint32_t k = rank_of(l);
      if (k >= limit || (shift < 24 && (k ^ found) >> (shift + 8))) return;
      const int b = (k >> shift) & 255;
      if (MASS) atomicAdd(&sh.mass[b], fixed(weight(r, l, sh.tab)));
      else atomicAdd(&sh.count[b], 1u);
    });
    lds_barrier();
    u64 before;
    const int b = MASS ? crossing<1>(sh.mass, target, before, sh) : crossing<1>(sh.count, target, before, sh);
    target -= before;
    found |= (uint32_t)b << shift;
  }
  if (!MASS)
    above = sum_of(src, sh, [&](int, float l) {
      return bin_of(r, l) == bin && rank_of(l) < found ? fixed(weight(r, l, sh.tab)) : 0;
    });
  return Cut{of_rank(found), target};
}

// The same among at most 64 elements, those that in() names: each is compared with all.
template <bool MASS, class S, class F>
__device__ __forceinline__ Cut cut_of_few(const Row &r, const S &src, F &&in, u64 target, u64 &above, Shared &sh) {
  const int t = threadIdx.x;
  lds_barrier();
  if (t == 0) sh.n = 0;
  lds_barrier();
  each(src, [&](int, float l) {
    if (!in(l)) return;
    const int i = atomicAdd(&sh.n, 1);
    sh.rank[i] = rank_of(l);
    sh.w[i] = fixed(weight(r, l, sh.tab));
  });
  lds_barrier();
  const int n = sh.n;
  if (t < n) {
    const uint32_t k = sh.rank[t];
    u64 wb = 0, wt = 0;
    uint32_t nb = 0, nt = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const uint32_t y = sh.rank[j];
      const u64 w = sh.w[j];
      wb += y < k ? w : 0;
      wt += y == k ? w : 0;
      nb += y < k;
      nt += y == k;
    }
    const u64 before = MASS ? wb : nb, here_ = MASS ? wt : nt;
    if (before < target && before + here_ >= target) {  // (equal ones write the same)
      sh.at = (int)k;
      sh.before = before;
      sh.above = wb;
    }
  }
  lds_barrier();
  above = sh.above;
  return Cut{of_rank((uint32_t)sh.at), target - sh.before};
}

// The same by the number of the bin's elements (`few` of them): up to 64 are compared with each
// other (`held`: the counts stay), more of a long row are gathered first.
template <bool MASS, bool FINER = true, class S>
__device__ __forceinline__ Cut cut_in_bin(const Row &r, const S &src, int bin, int few, uint32_t limit, u64 target,
                                          u64 &above, bool &held, Shared &sh) {
  const int t = threadIdx.x;
  if (few > 64) {
    held = false;
    if constexpr (std::is_same<S, Logits>::value) {
      if (few <= kCand) {
        lds_barrier();
        if (t == 0) sh.n = 0;
        lds_barrier();
        each(src, [&](int, float l) {
          if (bin_of(r, l) == bin) sh.cand[atomicAdd(&sh.n, 1)] = l;
        });
        lds_barrier();
        return cut_by_digits<MASS>(r, Candidates{sh.cand, sh.n}, bin, limit, target, above, sh);
      }
    }
    if constexpr (FINER && MASS && std::is_same<S, Candidates>::value) {
      // finer bins of what lies in this one (the others' elements fall in the first and the
      // last, which the cut is not looked for among)
      Row f = r;
      f.top = r.top - (float)bin / r.scale;
      f.scale = r.scale * kBins;
      auto in = [&](float l) { return bin_of(r, l) == bin && rank_of(l) < limit; };
      lds_barrier();
      clear(sh.mass);
      clear(sh.count);
      lds_barrier();
      each(src, [&](int, float l) {
        if (!in(l)) return;
        const int b = bin_of(f, l);
        atomicAdd(&sh.mass[b], fixed(weight(r, l, sh.tab)));
        atomicAdd(&sh.count[b], 1u);
      });
      lds_barrier();
      u64 before;
      const int b = crossing(sh.mass, target, before, sh);
      if (sh.count[b] <= 64) return cut_of_few<true>(r, src, [&](float l) { return in(l) && bin_of(f, l) == b; }, target - before, above, sh);
    }
    return cut_by_digits<MASS>(r, src, bin, limit, target, above, sh);
  }
  return cut_of_few<MASS>(r, src, [&](float l) { return bin_of(r, l) == bin && rank_of(l) < limit; }, target, above, sh);
}

// The first whole number that is p times x or more, 1 .. x's own.
__device__ __forceinline__ u64 part_of(float p, u64 x) {
  const double y = (double)p * (double)x;
  u64 n = (u64)y;
  n += (double)n < y;
  return n > 1 ? n : 1;
}

// The cut by top_k (src.n or more: none) and top_p (1 or more: none) among the elements. all_: the
// whole row's sum by its chunks (0: the elements' own), which top_p is a part of; the elements need not be the whole row.
template <class S>
__device__ __forceinline__ Cut find_cut(const Row &r, const S &src, int k, float p, u64 all_, Shared &sh) {
  Cut cut{-INFINITY, ~0ull};
  if (k >= src.n && p >= 1.0f) return cut;
  lds_barrier();
  clear(sh.mass);
  clear(sh.count);
  lds_barrier();
  each(src, [&](int, float l) {
    const int b = bin_of(r, l);
    atomicAdd(&sh.count[b], 1u);
    if (p < 1.0f) {
      const u64 w = fixed(weight(r, l, sh.tab));
      if (w) atomicAdd(&sh.mass[b], w);
    }
  });
  lds_barrier();
  // k falls into bin kb; m_bins: the sum of the bins before it, m_above: of all elements
  // before the k-th's value
  u64 n_before = 0, m_bins = 0, w_tie = 0;
  int kb = kBins;
  if (k < src.n) kb = crossing(sh.count, (u64)k, n_before, sh);
  if (p < 1.0f) m_bins = sum_below(sh.mass, kb, sh);
  u64 m_above = m_bins, all = m_bins, above;
  bool held = true;
  if (kb < kBins) {
    cut = cut_in_bin<false>(r, src, kb, (int)sh.count[kb], 0xffffffffu, (u64)k - n_before, above, held, sh);
    if (p >= 1.0f) return cut;
    w_tie = fixed(weight(r, cut.v, sh.tab));
    m_above += above;
    all = m_above + cut.ties * w_tie;
  }
  u64 target = part_of(p, all_ ? all_ : all);
  if (target > all) {
    if (all_) return cut;  // further down than the elements go
    target = all;
  }
  if (target > m_above) {
    cut.ties = (target - m_above + w_tie - 1) / w_tie;
    return cut;
  }
  u64 before = m_bins;
  int b = kb;
  uint32_t limit = rank_of(cut.v);
  if (target <= m_bins) {
    b = crossing(sh.mass, target, before, sh);
    limit = 0xffffffffu;
  }
  cut = cut_in_bin<true>(r, src, b, held ? (int)sh.count[b] : src.n, limit, target - before, above, held, sh);
  w_tie = fixed(weight(r, cut.v, sh.tab));
  cut.ties = (cut.ties + w_tie - 1) / w_tie;
  return cut;
}

// The first kept element at which the running sum passes u times the sum, or `goal` where `whole`
// is given (the sum of a row of which src is a part). More elements than kSegment: by
// the sums of segments first, a wave each. Returns its weight and the sum; -1 where all
// weights are 0.
template <class S>
__device__ __forceinline__ int draw(const Row &r, const S &src, const Cut &cut, u64 goal, u64 whole, u64 &w, u64 &sum,
                                    Shared &sh) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  auto kept = [&](float l) -> u64 {
    const double x = weight(r, l, sh.tab);
    return x >= r.min_w ? fixed(x) : 0;
  };
  const u64 w_tie = kept(cut.v);
  const bool limited = cut.ties < (u64)src.n;  // some of those equal to v may be left out
  int start = 0, len = src.n;
  u64 ties = cut.ties, total;
  auto begin = [&]() {
    sum = whole ? whole : total;
    if (!whole) goal = (u64)((double)r.u * (double)sum);
    goal = goal < total ? goal : total - 1;  // (a part's sum, as the row's was formed, may be some units off)
  };
  if (len > kSegment) {
    const int n = (len + kSegment - 1) / kSegment;
    lds_barrier();
    float x[kSegment / 64], next[kSegment / 64];
    auto load = [&](int k) {
      const int a = k * kSegment + lane;
#pragma unroll
      for (int j = 0; j < kSegment / 64; ++j) next[j] = src.l[a + j * 64 < len ? a + j * 64 : len - 1];
    };
    load(wave);
    for (int k = wave; k < n; k += kWaves) {
      const int a = k * kSegment + lane, b = k * kSegment + kSegment < len ? k * kSegment + kSegment : len;
      u64 s = 0;
      uint32_t c = 0;
#pragma unroll
      for (int j = 0; j < kSegment / 64; ++j) x[j] = clean(next[j]);
      if (k + kWaves < n) load(k + kWaves);
#pragma unroll
      for (int j = 0; j < kSegment / 64; ++j) {
        const u64 y = kept(x[j]);
        const bool in = a + j * 64 < b;
        s += in && (limited ? x[j] > cut.v : x[j] >= cut.v) ? y : 0;
        c += in && x[j] == cut.v;
      }
      s = wave_scan(s);
      if (limited) c = (uint32_t)group_sum_i<64>((int)c);
      if (lane == 63) {
        sh.mass[k] = s;
        if (limited) sh.count[k] = c;
      }
    }
    lds_barrier();
    u64 s[kBinsEach], all = 0, mine = 0, held = 0;
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e) s[e] = kBinsEach * t + e < n ? sh.mass[kBinsEach * t + e] : 0;
    if (limited) {  // how many of the equal ones each segment keeps
      uint32_t c[kBinsEach];
      u64 x = 0;
#pragma unroll
      for (int e = 0; e < kBinsEach; ++e) x += c[e] = kBinsEach * t + e < n ? sh.count[kBinsEach * t + e] : 0;
      held = block_scan(x, total, sh);
      u64 before = held;
#pragma unroll
      for (int e = 0; e < kBinsEach; ++e) {
        const u64 left = ties > before ? ties - before : 0;
        s[e] += (c[e] < left ? c[e] : left) * w_tie;
        before += c[e];
      }
    }
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e) mine += s[e];
    all = block_scan(mine, total, sh);
    if (!total) return -1;
    begin();
    if (all <= goal && goal < all + mine) {
      int e = 0;
#pragma unroll
      for (int k = 0; k < kBinsEach - 1; ++k)
        if (e == k && all + s[k] <= goal) {
          all += s[k];
          if (limited) held += sh.count[kBinsEach * t + k];
          ++e;
        }
      sh.at = kBinsEach * t + e;
      sh.before = all;
      sh.ties = held;
    }
    lds_barrier();
    start = sh.at * kSegment;
    len = start + kSegment < len ? kSegment : len - start;
    goal -= sh.before;
    ties = limited ? (ties > sh.ties ? ties - sh.ties : 0) : ties;
    lds_barrier();
  }
  // EACH elements a thread
  constexpr int EACH = kSegment / kThreads;
  float l[EACH];
  u64 m[EACH], x = 0, nth = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) l[e] = EACH * t + e < len ? src.at(start + EACH * t + e) : -INFINITY;
  if (limited) {
#pragma unroll
    for (int e = 0; e < EACH; ++e) x += EACH * t + e < len && l[e] == cut.v;
    nth = block_scan(x, total, sh);
    x = 0;
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const bool in = EACH * t + e < len, tie = in && l[e] == cut.v;
    x += m[e] = in && (l[e] > cut.v || (tie && (!limited || nth < ties))) ? kept(l[e]) : 0;
    nth += tie;
  }
  u64 at = block_scan(x, total, sh);
  if (src.n <= kSegment) {
    if (!total) return -1;
    begin();
  }
  if (at <= goal && goal < at + x) {
    int e = 0;
#pragma unroll
    for (int k = 0; k < EACH - 1; ++k)
      if (e == k && at + m[k] <= goal) {
        at += m[k];
        ++e;
      }
    u64 v = 0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) v = e == k ? m[k] : v;
    sh.at = start + EACH * t + e;
    sh.before = v;
  }
  lds_barrier();
  w = sh.before;
  return sh.at;
}

}  // namespace

// A row that work-groups share: its cut lies in `bin`, where target is left of what is
// looked for; the parts' sums before it.
struct SampleRow {
  float top, scale;
  int shared, bin;  // shared: work-groups, 0: the row is done
  unsigned long long target;
  unsigned long long part[kParts];
};

namespace {

// Chunks of a row in the workspace: whole fours.
__host__ __device__ __forceinline__ int chunk_stride(int chunks) { return (chunks + 3) & ~3; }

// A row's settings, as they are used.
struct Settings {
  float temp, p, min_p;
  int k;
  bool greedy;
  __device__ __forceinline__ Settings(const SampleArgs &a, int64_t row) {
    temp = a.temperature ? a.temperature[row] : 1.0f;
    k = a.top_k ? a.top_k[row] : 0;
    k = k > 0 && k < (int)a.n ? k : (int)a.n;
    p = a.top_p ? a.top_p[row] : 1.0f;
    p = p == p ? p : 1.0f;
    min_p = a.min_p ? a.min_p[row] : 0.0f;
    min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
    greedy = !(temp > 0.0f) || k == 1 || p <= 0.0f;
  }
  __device__ __forceinline__ Row row(float top, float u) const {
    Row r;
    r.top = top;
    r.max = top;
    r.inv_t = fmax(369.32993046757463 / (double)temp, 1e-300);  // (T = inf: all finite logits weigh the same)
    r.min_w = (double)min_p * 0x1p43;
    r.u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    return r;
  }
  // Bins per unit of logit; low: the lowest one.
  __device__ __forceinline__ float scale(float top, float low, bool weights) const {
    return fminf(fmaxf((kBins - 1) / fminf(top - low, (weights ? 0.0f : kSpan) + kSpanT * temp), 1.0e-37f), 3.0e38f);
  }
  // whether the sum of all weights is asked for
  __device__ __forceinline__ bool sums(const SampleArgs &a) const { return !greedy && k >= (int)a.n && (p < 1.0f || min_p == 0.0f); }
};

// Per chunk of kChunk logits, the largest, the sum of the weights by that one (kFix
// units) where it is asked for, and the largest of every kGroup. A wave takes `each`
// chunks one after the other, the next one's loads on their way meanwhile, and waits for
// no other wave. Bound by the vector units where sums are asked for (32 instructions a logit, 20 of
// them the weight's, 14 in 64 bits: 256 rows of 151936 46 us, 3.4 TB/s), otherwise by the loads (30).
__global__ void __launch_bounds__(256) k_sample_stats(SampleArgs a, int64_t row0, SampleStats st, int chunks, int each) {
  constexpr int U = kChunk / 256;
  __shared__ double tab[kTab];
  const int t = threadIdx.x, lane = t & 63, c0 = (blockIdx.x * 4 + (t >> 6)) * each;
  const int c1 = c0 + each < chunks ? c0 + each : chunks;
  const int64_t row = row0 + blockIdx.y;
  const float *l = a.logits + row * a.stride;
  const int n = (int)a.n;
  float next[U][4];
  auto load = [&](int c) {
    const int base = c * kChunk + 4 * lane;
    if (c * kChunk + kChunk <= n) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const f32x4a4 y = *(const f32x4a4 *)(l + base + j * 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) next[j][e] = y[e];
      }
    } else {
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) next[j][e] = base + j * 256 + e < n ? l[base + j * 256 + e] : -INFINITY;
    }
  };
  if (c0 < c1) load(c0);
  const Settings s(a, row);
  const bool sums = s.sums(a);
  if (sums) {
    make_table(tab);
    lds_barrier();
  }
  for (int c = c0; c < c1; ++c) {
    float x[U][4];
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = clean(next[j][e]);
    if (c + 1 < c1) load(c + 1);
    const int64_t at = (int64_t)blockIdx.y * chunk_stride(chunks) + c;
    float *gm = st.group_max + at * (kChunk / kGroup);
    float m = -INFINITY, low = INFINITY;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float g = max2(max2(x[j][0], x[j][1]), max2(x[j][2], x[j][3]));
      g = max2(g, dpp_f<kDppXor1>(g));
      g = max2(g, dpp_f<kDppXor2>(g));
      g = max2(g, dpp_f<kDppHalfMirror>(g));
      g = max2(g, dpp_f<kDppMirror>(g));
      if ((lane & 15) == 0) gm[j * 4 + (lane >> 4)] = g;
      m = max2(m, g);
      low = fminf(low, g == -INFINITY ? INFINITY : g);
    }
    m = max2(m, __shfl_xor(m, 16));
    m = max2(m, __shfl_xor(m, 32));
    low = fminf(low, __shfl_xor(low, 16));
    low = fminf(low, __shfl_xor(low, 32));
    u64 sum = 0;
    if (sums) {
      const Row r = s.row(m, 0.0f);
      auto add = [&](auto inf_) {
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)  // (-inf, past the row's end, weighs nothing)
            sum += (u64)__double_as_longlong(weight<decltype(inf_)::value>(r, x[j][e], tab) + 0x1p52);
        sum -= (u64)(4 * U) * 0x4330000000000000ull;  // (the sum's exponents, see fixed())
      };
      if (m == INFINITY) add(std::true_type());
      else add(std::false_type());
      sum = wave_scan(sum);
    }
    if (lane == 63) {
      st.chunk_max[at] = m;
      st.chunk_low[at] = low;
      st.chunk_sum[at] = sum;
    }
  }
}

// The first element of [start, end) that is l.
__device__ __forceinline__ int first_equal(const Logits &src, int start, int end, float l, Shared &sh) {
  lds_barrier();
  if (threadIdx.x == 0) sh.at = end;
  lds_barrier();
  int first = end;
  for (int i = start + threadIdx.x; i < end && first == end; i += 4 * kThreads) {
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = src.at(i + j * kThreads < end ? i + j * kThreads : i);
#pragma unroll
    for (int j = 3; j >= 0; --j) first = x[j] == l && i + j * kThreads < end ? i + j * kThreads : first;
  }
  if (first < end) atomicMin(&sh.at, first);
  lds_barrier();
  return sh.at;
}

// The largest of a thread's four groups from g on (16-byte aligned).
__device__ __forceinline__ f32x4a4 groups_at(const float *gm, int n_group, int g) {
  f32x4a4 x = *(const f32x4a4 *)(gm + (g < n_group ? g : 0));  // (a chunk's groups, beyond the row's too, are all written)
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = g + e < n_group ? x[e] : -INFINITY;
  return x;
}

// Candidates of sh.group's n groups, in their order, behind the first `have`; a row of 16
// lanes per group, U of them at a time. Returns how many there are now (they end at kCand).
template <int U>
__device__ __forceinline__ int gather_groups(const Row &r, const Logits &src, int n, int b0, Shared &sh) {
  constexpr int ROWS = kThreads / 16;
  static_assert(U * ROWS <= 128, "two counts a lane");
  const int t = threadIdx.x, l16 = t & 15, lane = t & 63;
  int have = 0;
  for (int i0 = 0; i0 < n && have <= kCand; i0 += U * ROWS) {
    float x[U][4];
    uint32_t in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * ROWS + (t >> 4), at = i < n ? sh.group[i] * kGroup + 4 * l16 : src.n;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[u][e] = src.l[at + e < src.n ? at + e : src.n - 1];
      in[u] = at + 4 <= src.n ? 15 : at < src.n ? (1u << (src.n - at)) - 1 : 0;
    }
    lds_barrier();  // (the last round's counts are read)
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[u][e] = clean(x[u][e]);
        if (x[u][e] == -INFINITY || bin_of(r, x[u][e]) > b0) in[u] &= ~(1u << e);
      }
      const int m = group_sum_i<16>(__builtin_popcount(in[u]));
      if (l16 == 0) sh.in_group[u * ROWS + (t >> 4)] = (uint16_t)m;
    }
    lds_barrier();
    // candidates before each of the round's groups, two a lane: every wave for itself
    const u64 c0 = 2 * lane < U * ROWS ? sh.in_group[2 * lane] : 0, c1 = 2 * lane < U * ROWS ? sh.in_group[2 * lane + 1] : 0;
    const int sum = (int)wave_scan(c0 + c1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = u * ROWS + (t >> 4), own = __builtin_popcount(in[u]);
      // up to the group's pair, without the pair's second where the group is the first
      int to = have + __shfl(sum, k >> 1) - (k & 1 ? sh.in_group[k] : sh.in_group[k] + sh.in_group[k + 1]);
      int before = own;  // inclusive, over the row of lanes
      before += __builtin_amdgcn_update_dpp(0, before, 0x111, 0xf, 0xf, false);
      before += __builtin_amdgcn_update_dpp(0, before, 0x112, 0xf, 0xf, false);
      before += __builtin_amdgcn_update_dpp(0, before, 0x114, 0xf, 0xf, false);
      before += __builtin_amdgcn_update_dpp(0, before, 0x118, 0xf, 0xf, false);
      to += before - own;
      const int first = i0 + k < n ? sh.group[i0 + k] * kGroup + 4 * l16 : 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (in[u] & (1u << e)) {
          if (to < kCand) {
            sh.cand[to] = x[u][e];
            sh.index[to] = first + e;
          }
          ++to;
        }
    }
    have += __shfl(sum, 63);
  }
  lds_barrier();
  return have;
}

// The elements whose even bin is at most b0, in sh.cand and sh.index, in their order;
// -1 where they are too many, or lie in more than `most` groups. A group's largest
// says whether it has any; g4: those of the thread's first groups.
__device__ __forceinline__ int gather(const Row &r, const Logits &src, const float *gm, f32x4a4 g4, int n_group, int b0, int most,
                                      Shared &sh) {
  const int t = threadIdx.x;
  int n = 0;
  for (int g0 = 0; g0 < n_group; g0 += 4 * kThreads) {
    const int g = g0 + 4 * t;
    if (g0) g4 = groups_at(gm, n_group, g);
    uint32_t in = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (g4[e] != -INFINITY && bin_of(r, g4[e]) <= b0) in |= 1u << e;
    u64 total;
    int at = n + (int)block_scan(__builtin_popcount(in), total, sh);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (in >> e & 1) {
        if (at < kGroups) sh.group[at] = (uint16_t)(g + e);
        ++at;
      }
    n += (int)total;
  }
  if (n > most) return -1;
  lds_barrier();
  n = n <= 64 ? gather_groups<4>(r, src, n, b0, sh) : gather_groups<8>(r, src, n, b0, sh);
  return n <= kCand ? n : -1;
}

// A row of which more is kept than fits the candidates, without top_k, is shared by work-groups,
// a part each. k_sample sums the weights of the parts by bins; the last work-group to
// arrive finds the bin that the target falls into. k_sample_shared gathers that bin's
// elements; the last to arrive finds the cut among them, and by the parts' sums the part
// that the drawn token is in, so that only that one is gone through.
__device__ __forceinline__ int part_len(int n, int parts) { return (n + parts - 1) / parts; }
__device__ __forceinline__ Logits part_at(const Logits &src, int len, int i) {
  const int a = i * len < src.n ? i * len : src.n;
  return Logits{src.l + a, src.n - a < len ? src.n - a : len};
}

// Whether this work-group is the last of `parts` to arrive. What is handed over is
// written and read by agent-scope accesses, which go past the XCDs' caches, and each
// wave has waited for its stores before the counter's add: no release besides.
__device__ __forceinline__ bool last_of(uint32_t *counter, int parts, Shared &sh) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.n = (int)__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (sh.n == parts - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return sh.n == parts - 1;
}

// The part that the drawn token is in by the parts' sums (sh.part), what is left of the
// goal there, and the sum.
__device__ __forceinline__ int part_drawn(const Row &r, int parts, u64 &goal, u64 &sum, const Shared &sh) {
  sum = 0;
  for (int k = 0; k < parts; ++k) sum += sh.part[k];
  goal = (u64)((double)r.u * (double)sum);
  goal = goal < sum ? goal : sum - 1;
  int k = 0;
  for (; k < parts - 1 && goal >= sh.part[k]; ++k) goal -= sh.part[k];
  return k;
}

// k_sample's share of that. With min_p what weighs that much is summed, too: where it is less
// than top_p asks for (or top_p asks for nothing) it is what is kept, and the last work-group to arrive
// draws. Returns the token then, otherwise -1. all_: the row's sum, as the chunks' say.
__device__ __forceinline__ int share(const Row &r, const Logits &src, float p, u64 all_, const SampleStats &st, int parts, u64 &w,
                                     u64 &sum, Shared &sh) {
  const int t = threadIdx.x, mine = blockIdx.y, len = part_len(src.n, parts);
  const bool bins = p < 1.0f, least = r.min_w > 0.0;
  lds_barrier();
  clear(sh.mass);
  lds_barrier();
  u64 heavy = 0;
  each(part_at(src, len, mine), [&](int, float l) {
    const double y = weight(r, l, sh.tab);
    const u64 x = fixed(y);
    if (least) heavy += y >= r.min_w ? x : 0;
    if (bins && x) atomicAdd(&sh.mass[bin_of(r, l)], x);
  });
  SampleRow *row = st.rows + blockIdx.x;
  if (least) {
    u64 total;
    block_scan(heavy, total, sh);
    if (t == 0) __hip_atomic_store(row->part + mine, total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  lds_barrier();
  u64 *all = st.part_sum + (int64_t)blockIdx.x * parts * kBins;
  if (bins)
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e)
      __hip_atomic_store(all + mine * kBins + e * kThreads + t, sh.mass[e * kThreads + t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (!last_of(st.counters + 2 * blockIdx.x, parts, sh)) return -1;
  u64 all_heavy = ~0ull;
  if (least) {
    if (t < parts) sh.part[t] = __hip_atomic_load(row->part + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    lds_barrier();
    all_heavy = 0;
    for (int k = 0; k < parts; ++k) all_heavy += sh.part[k];
  }
  u64 target = ~0ull, before = 0;
  int b = 0;
  if (bins) {
    u64 s[kBinsEach] = {};
    for (int k0 = 0; k0 < parts; k0 += 8) {
      u64 x[8][kBinsEach];
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < kBinsEach; ++e)
          x[k][e] = k0 + k < parts ? __hip_atomic_load(all + (k0 + k) * kBins + e * kThreads + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < kBinsEach; ++e) s[e] += x[k][e];
    }
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e) sh.mass[e * kThreads + t] = s[e];
    lds_barrier();
    const u64 total = sum_below(sh.mass, kBins, sh);
    target = part_of(p, all_);
    target = target < total ? target : total;
    b = crossing(sh.mass, target, before, sh);
  }
  if (all_heavy < target) {
    u64 goal;
    const int k = part_drawn(r, parts, goal, sum, sh);
    return k * len + draw(r, part_at(src, len, k), Cut{-INFINITY, ~0ull}, goal, sum, w, sum, sh);
  }
  if (t == 0) {
    row->top = r.top;
    row->scale = r.scale;
    row->shared = parts;
    row->bin = b;
    row->target = target - before;
  }
  return -1;
}

__device__ __forceinline__ void answer(const SampleArgs &a, int64_t row, int id, float prob) {
  a.out[row] = (uint32_t)id;
  if (a.prob) a.prob[row] = prob;
  if (a.pos) a.pos[row] += a.advance;
}

// Bound by latencies, too (16 flat rows 23 us: the part's elements 7, the hand-over, the cut
// among the bin's, a part's draw). Grid: (rows, parts).
__global__ void __launch_bounds__(kThreads) k_sample_shared(SampleArgs a, int64_t row0, SampleStats st) {
  const SampleRow *have = st.rows + blockIdx.x;
  const int parts = have->shared;
  if (parts == 0) return;
  __shared__ Shared sh;
  const int t = threadIdx.x;
  const int64_t row = row0 + blockIdx.x;
  make_table(sh.tab);
  if (t == 0) sh.n = 0;
  lds_barrier();
  const Logits src{a.logits + row * a.stride, (int)a.n};
  Row r = Settings(a, row).row(have->top, a.u[row]);
  r.scale = have->scale;
  const int len = part_len(src.n, parts), mine = blockIdx.y, b = have->bin;
  each(part_at(src, len, mine), [&](int i, float l) {
    if (bin_of(r, l) != b) return;
    const int k = atomicAdd(&sh.n, 1);
    if (k < kCand) {
      sh.cand[k] = l;
      sh.index[k] = mine * len + i;
    }
  });
  lds_barrier();
  // the part's sum before the bin
  u64 *all = st.part_sum + ((int64_t)blockIdx.x * parts + mine) * kBins, s = 0, below;
#pragma unroll
  for (int e = 0; e < kBinsEach; ++e) {
    const u64 x = __hip_atomic_load(all + e * kThreads + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s += e * kThreads + t < b ? x : 0;
  }
  block_scan(s, below, sh);
  uint32_t *const counter = st.counters + 2 * blockIdx.x;
  unsigned long long *const part = st.rows[blockIdx.x].part;
  if (t == 0) __hip_atomic_store(part + mine, below, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  u64 *list = st.in_bin + (int64_t)blockIdx.x * kCand;
  const int own = sh.n;
  if (t == 0) sh.at = (int)__hip_atomic_fetch_add(counter + 1, (uint32_t)own, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  lds_barrier();
  const int at = sh.at;
  for (int i = t; i < own && i < kCand && at + i < kCand; i += kThreads)
    __hip_atomic_store(list + at + i, (u64)(uint32_t)sh.index[i] << 32 | __float_as_uint(sh.cand[i]), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  if (!last_of(counter, parts, sh)) return;
  const int n = (int)__hip_atomic_load(counter + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int i = t; i < n && i < kCand; i += kThreads) {
    const u64 x = __hip_atomic_load(list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh.cand[i] = __uint_as_float((uint32_t)x);
    sh.index[i] = (int)(x >> 32);
  }
  __syncthreads();
  if (t == 0) __hip_atomic_store(counter + 1, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  u64 none, w, sum;
  bool held = true;
  Cut cut = n > kCand ? cut_by_digits<true>(r, src, b, 0xffffffffu, have->target, none, sh)
                      : cut_in_bin<true>(r, Candidates{sh.cand, n}, b, n, 0xffffffffu, have->target, none, held, sh);
  const u64 w_tie = fixed(weight(r, cut.v, sh.tab));
  cut.ties = (cut.ties + w_tie - 1) / w_tie;
  // the parts' sums, where none of the equal ones is left out (all of the kept weigh min_p)
  u64 equal = 0;
  if (n <= kCand) {
    lds_barrier();
    if (t < parts) sh.part[t] = __hip_atomic_load(part + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    lds_barrier();
    uint32_t c = 0;
    for (int i = t; i < n; i += kThreads) {
      const float l = sh.cand[i];
      c += l == cut.v;
      if (l >= cut.v) atomicAdd(&sh.part[sh.index[i] / len], fixed(weight(r, l, sh.tab)));
    }
    block_scan(c, equal, sh);
  }
  int id;
  if (n > kCand || equal > cut.ties) {
    id = draw(r, src, cut, 0, 0, w, sum, sh);
  } else {
    u64 goal;
    const int k = part_drawn(r, parts, goal, sum, sh);
    id = k * len + draw(r, part_at(src, len, k), Cut{cut.v, ~0ull}, goal, sum, w, sum, sh);
  }
  if (t == 0) answer(a, row, id, (float)((double)w / (double)sum));
}

// A row by what k_sample_stats found. A chain of short steps, bound by their latencies: a row
// without a cut 6 us, top_k 40 and top_p 0.95 of 32000 tokens 13, a flat row's bins 18.
// chunks: 0 without k_sample_stats before it. Grid: (rows, work-groups that may share one).
__global__ void __launch_bounds__(kThreads) k_sample(SampleArgs a, int64_t row0, SampleStats st, int chunks) {
  __shared__ Shared sh;
  const int t = threadIdx.x;
  const int64_t row = row0 + blockIdx.x;
  const Settings s(a, row);
  const bool flat = gridDim.y > 1 && !s.greedy && s.k >= (int)a.n && (s.p < 1.0f || s.min_p > 0.0f);  // (the others are one work-group's)
  if (blockIdx.y && !flat) return;
  make_table(sh.tab);
  const Logits src{a.logits + row * a.stride, (int)a.n};
  // the largest logit, and the lowest of the groups' largest (without groups: of all)
  float m = -INFINITY, low = INFINITY;
  const int64_t c0 = (int64_t)blockIdx.x * chunk_stride(chunks);
  const float *gm = st.group_max + c0 * (kChunk / kGroup);
  const int n_group = (src.n + kGroup - 1) / kGroup;
  f32x4a4 g4{0};
  constexpr int CE = 4;  // chunks a thread, at most KMOE_SAMPLE_MAX / kChunk in all
  u64 chunk_sum[CE] = {};
  float chunk_max[CE];
#pragma unroll
  for (int e = 0; e < CE; ++e) chunk_max[e] = -INFINITY;
  if (chunks) {
    g4 = groups_at(gm, n_group, 4 * t);
    if (CE * t < chunks) {
#pragma unroll
      for (int e = 0; e < CE; ++e) {  // (whole fours are there, those past the row's are not looked at)
        const bool in = CE * t + e < chunks;
        const float x = st.chunk_max[c0 + CE * t + e], y = st.chunk_low[c0 + CE * t + e];
        const u64 z = st.chunk_sum[c0 + CE * t + e];
        chunk_max[e] = in ? x : -INFINITY;
        chunk_sum[e] = in ? z : 0;
        m = fmaxf(m, chunk_max[e]);
        low = fminf(low, in ? y : INFINITY);
      }
    }
  } else {
    each(src, [&](int, float l) {
      m = fmaxf(m, l);
      low = fminf(low, l == -INFINITY ? INFINITY : l);
    });
  }
  m = group_max<64>(m);
  low = -group_max<64>(-low);
  if ((t & 63) == 0) {
    sh.redf[0][t >> 6] = m;
    sh.redf[1][t >> 6] = low;
  }
  lds_barrier();
  for (int i = 0; i < kWaves; ++i) {
    m = fmaxf(m, sh.redf[0][i]);
    low = fminf(low, sh.redf[1][i]);
  }
  Row r = s.row(m, a.u[row]);
  r.scale = s.scale(m, low, false);
  int id = 0;
  float prob = 0.0f;
  if (m == -INFINITY) {  // nothing to draw from
    if (blockIdx.y) return;
  } else if (s.greedy) {
    int start = 0, end = src.n;
    if (chunks) {
      if (t == 0) sh.at = chunks;
      lds_barrier();
#pragma unroll
      for (int e = 0; e < CE; ++e)
        if (chunk_max[e] == m) atomicMin(&sh.at, CE * t + e);
      lds_barrier();
      start = sh.at * kChunk;
      end = start + kChunk < end ? start + kChunk : end;
    }
    id = first_equal(src, start, end, m, sh);
    prob = 1.0f;
  } else {
    // the chunks' sums by the row's largest
    u64 sum = 0, w = 0, mine = 0, before = 0;
    if (chunks && s.sums(a)) {
#pragma unroll
      for (int e = 0; e < CE; ++e) {
        // (nothing where not even the largest weighs a unit: no token of it can be drawn. Where it
        // does, so does the sum: both are rounded alike)
        const double y = weight(r, chunk_max[e], sh.tab);
        chunk_sum[e] = fixed(y) ? (u64)__builtin_rint((double)chunk_sum[e] * 0x1p-43 * y) : 0;
        mine += chunk_sum[e];
      }
      before = block_scan(mine, sum, sh);
    }
    int at = -1;
    if (sum && s.p >= 1.0f) {  // everything is kept: the chunk, then the token in it
      u64 goal = (u64)((double)r.u * (double)sum);
      goal = goal < sum ? goal : sum - 1;
      if (before <= goal && goal < before + mine) {
        int e = 0;
#pragma unroll
        for (int k = 0; k < CE - 1; ++k)
          if (e == k && before + chunk_sum[k] <= goal) {
            before += chunk_sum[k];
            ++e;
          }
        sh.at = CE * t + e;
        sh.before = before;
      }
      lds_barrier();
      const int start = sh.at * kChunk, end = start + kChunk < src.n ? start + kChunk : src.n;
      // (the chunk's sum may be less than those of its tokens, of which u = 1 finds the last)
      goal = r.u < 1.0f ? goal - sh.before : ~0ull;
      lds_barrier();
      at = draw(r, Logits{src.l + start, end - start}, Cut{-INFINITY, ~0ull}, goal, sum, w, sum, sh);
      id = start + at;
    } else if (chunks) {
      // a bin that holds the last kept token, or one after it, by the groups' largest: as
      // many of them as tokens are kept, or of as much weight
      int b0 = kBins;
      lds_barrier();
      if (s.k < src.n) clear(sh.count);
      else clear(sh.mass);
      lds_barrier();
      for (int g = 4 * t; g < n_group; g += 4 * kThreads) {
        const f32x4a4 y = g < 4 * kThreads ? g4 : groups_at(gm, n_group, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (y[e] == -INFINITY) continue;
          const int b = bin_of(r, y[e]);
          if (s.k < src.n) atomicAdd(&sh.count[b], 1u);
          else if (s.p < 1.0f) atomicAdd(&sh.mass[b], fixed(weight(r, y[e], sh.tab)));
        }
      }
      lds_barrier();
      u64 total, none;
      if (s.k < src.n) {
        total = sum_below(sh.count, kBins, sh);
        if ((u64)s.k <= total) b0 = crossing(sh.count, (u64)s.k, none, sh);
      } else if (s.p < 1.0f) {
        const u64 target = part_of(s.p, sum);
        total = sum_below(sh.mass, kBins, sh);
        if (target <= total) b0 = crossing(sh.mass, target, none, sh);
      }
      if (s.min_p > 0.0f && (s.k >= src.n || s.p >= 1.0f)) {
        // (where top_p counts among the top_k all of those are needed)
        const float x = (float)(-log((double)s.min_p) * (double)s.temp) * r.scale + 1.0f;
        b0 = x < (float)b0 ? (int)x : b0;
      }
      if (b0 < kBins - 1) {
        // (a row that may be shared is, rather than going through more groups than this: 256
        // took 6 us, 1000 20)
        const int n = gather(r, src, gm, g4, n_group, b0, flat ? kFewGroups : kGroups, sh);
        if (n >= 0) {
          if (blockIdx.y) return;
          const Candidates cand{sh.cand, n};
          Row f = r;
          f.scale = r.scale * ((float)kBins / (float)(b0 + 1));  // (their bins, finer)
          const Cut cut = find_cut(f, cand, s.k, s.p, s.k < src.n ? 0 : sum, sh);
          at = draw(f, cand, cut, 0, 0, w, sum, sh);
          id = sh.index[at];
        }
      }
    }
    if (at < 0) {
      // (elements lie about as far below the groups' largest as those lie apart, twice or three times)
      r.scale = s.scale(m, chunks ? m - 4.0f * (m - low) - 1.0f : low, s.k >= src.n);
      if (flat) {
        id = share(r, src, s.p, sum, st, (int)gridDim.y, w, sum, sh);
        if (id < 0) return;
      } else {
        const Cut cut = find_cut(r, src, s.k, s.p, s.k < src.n ? 0 : sum, sh);
        id = draw(r, src, cut, 0, 0, w, sum, sh);
      }
    }
    prob = (float)((double)w / (double)sum);
  }
  if (t == 0) {
    answer(a, row, id, prob);
    if (gridDim.y > 1) st.rows[blockIdx.x].shared = 0;
  }
}

constexpr int64_t kFewTokens = 8192;  // a work-group reads so many as quickly as another launch comes
// Rows times the work-groups that share one, and the tokens from which rows are shared: it takes
// another launch (4 us), whether a row turns out to be kept for the most part or not.
constexpr int kShareRows = 512;
constexpr int64_t kShareTokens = 65536;
constexpr size_t kStatBytes = (size_t)16 << 20, kSumBytes = (size_t)kShareRows * kBins * 8,
                 kListBytes = (size_t)kShareRows / 2 * kCand * 8, kRowBytes = kShareRows / 2 * sizeof(SampleRow);

}  // namespace

size_t sample_ws_bytes() { return kStatBytes + kSumBytes + kListBytes + kRowBytes; }
int sample_counters() { return kShareRows; }

hipError_t launch_sample(hipStream_t st, const SampleArgs &a, uint8_t *ws, uint32_t *counters) {
  if (a.n <= kFewTokens) {
    KMOE_LAUNCH(k_sample, dim3((unsigned)a.rows), dim3(kThreads), 0, st, a, (int64_t)0, SampleStats{}, 0);
    return hipGetLastError();
  }
  const int chunks = (int)((a.n + kChunk - 1) / kChunk), stride = chunk_stride(chunks);
  const int64_t bytes = (int64_t)stride * (16 + 4 * (kChunk / kGroup)), most = (int64_t)kStatBytes / bytes;
  for (int64_t row = 0; row < a.rows; row += most) {
    const int64_t n = a.rows - row < most ? a.rows - row : most;
    // the chip's work-groups among few rows that top_p may leave much of
    int parts = (a.top_p || a.min_p) && a.n >= kShareTokens && n <= kShareRows / 2 ? (int)(kShareRows / n) : 1;
    parts = parts < kParts ? parts : kParts;
    auto at = [&](int64_t x) { return (float *)(ws + x * most * stride); };
    uint8_t *const sums = ws + kStatBytes, *const list = sums + kSumBytes;
    const SampleStats s{(unsigned long long *)ws,   at(8), at(12), at(16), (unsigned long long *)sums, (SampleRow *)(list + kListBytes),
                        (unsigned long long *)list, counters};
    // chunks a wave: one where the waves do not fill the chip four times, at most eight
    const int64_t fill = n * chunks / 4096;
    const int each = fill < 1 ? 1 : fill < 8 ? (int)fill : 8;
    KMOE_LAUNCH(k_sample_stats, dim3((unsigned)(chunks + 4 * each - 1) / (4 * each), (unsigned)n), dim3(256), 0, st, a, row, s, chunks, each);
    KMOE_LAUNCH(k_sample, dim3((unsigned)n, (unsigned)parts), dim3(kThreads), 0, st, a, row, s, chunks);
    if (parts > 1 && a.top_p) KMOE_LAUNCH(k_sample_shared, dim3((unsigned)n, (unsigned)parts), dim3(kThreads), 0, st, a, row, s);
  }
  return hipGetLastError();
}

}  // namespace kmoe
