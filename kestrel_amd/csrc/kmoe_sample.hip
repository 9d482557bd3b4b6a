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
// step of u) in all.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "kmoe_device.h"
#include "kmoe_launch.h"

namespace kmoe {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kFix = 43;    // weights in units of 2^-43
constexpr int kBins = 2048;
constexpr int kTab = 256;
constexpr int kGroup = 64, kChunk = 4096;  // elements of which k_sample_stats finds the largest, and the sum
constexpr int kCand = 2048, kGroups = 1024;
constexpr int kFew = 1024;  // elements of a bin that are compared one with another
constexpr int kParts = 8;   // work-groups that share a row at most
// Distances from the largest logit that the even bins tell apart: to the lowest that is binned,
// at most this (a mask's -10^9 is none of the others' business) and 24 T, where
// weights are what counts 24 T.
constexpr float kSpan = 64.0f, kSpanT = 24.0f;

// NaN as -inf. Order of the logits as whole numbers: the larger the logit, the smaller
// its rank (-0 as 0).
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }
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
  if (threadIdx.x < kTab) tab[threadIdx.x] = exp2((double)threadIdx.x / kTab);
}

// A weight in units: z = 256 log2 of it is i + f, |f| <= 1/2, and 2^(z / 256) a power of two
// times 2^((i mod 256) / 256) (LDS) times the exponential of f log(2) / 256 by its
// series, whose fifth power's term is 2^-54.5. i comes out of z's sum with 1.5 2^52,
// whose last bit is 1. The largest logit's weight is 2^43 exactly. Below 2^-44 (-31
// nats: z = -11450) the weight rounds to no unit, whatever it is. A NaN is an infinite
// largest logit's distance from itself.
__device__ __forceinline__ double weight(const Row &r, float l, const double *tab) {
  double z = ((double)l - r.max) * r.inv_t;
  z = fmax(fmin(z, 0.0), -11450.0);
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
  float redf[3][kWaves];
  u64 part[kParts];
  u64 before, above;
  int at, n;
  // elements of one bin
  uint32_t rank[64];
  u64 w[64];
  // candidates, and the groups that they are in with how many candidates each has
  float cand[kCand];
  int index[kCand];
  uint16_t group[kGroups], in_group[kGroups];
};

// Inclusive scan over a wave: within rows of 16 lanes, then row 0's and 2's totals onto
// rows 1 and 3, then lane 31's onto the upper half.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_add(u64 x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xf, false);
  return x + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 wave_scan(u64 x) {
  x = dpp_add<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // row_bcast 15, 31
  return dpp_add<0x143, 0xc>(x);
}
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

// The first bin at which the running sum of hist reaches `target` (1 .. the total), and
// the sum before it.
template <class T>
__device__ __forceinline__ int crossing(const T *hist, u64 target, u64 &before, Shared &sh) {
  const int t = threadIdx.x;
  const u64 a = hist[2 * t], b = hist[2 * t + 1];
  u64 total;
  const u64 x = block_scan(a + b, total, sh);
  if (x < target && x + a + b >= target) {
    const bool second = x + a < target;
    sh.at = 2 * t + second;
    sh.before = x + (second ? a : 0);
  }
  lds_barrier();
  before = sh.before;
  return sh.at;
}

// f(i, l) for every element i, a work-group together.
template <class S, class F>
__device__ __forceinline__ void each(const S &src, F &&f) {
  constexpr int U = 8;
  int i = threadIdx.x;
  for (; i + (U - 1) * kThreads < src.n; i += U * kThreads) {
    float x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) x[j] = src.at(i + j * kThreads);
#pragma unroll
    for (int j = 0; j < U; ++j) f(i + j * kThreads, x[j]);
  }
  for (; i < src.n; i += kThreads) f(i, src.at(i));
}

template <class T>
__device__ __forceinline__ void clear(T *h) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) h[i] = 0;
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
  for (int d = 0; d < 3; ++d) {  // 11, 11 and 10 bits
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, top = d == 0 ? 32 : d == 1 ? 21 : 10;
    lds_barrier();
    if (MASS) clear(sh.mass);
    else clear(sh.count);
    lds_barrier();
    each(src, [&](int, float l) {
      if (bin_of(r, l) != bin) return;
      const uint32_t k = rank_of(l);
      if (k >= limit || (d && k >> top != found >> top)) return;
      const int b = (k >> shift) & (d == 2 ? 1023 : 2047);
      if (MASS) atomicAdd(&sh.mass[b], fixed(weight(r, l, sh.tab)));
      else atomicAdd(&sh.count[b], 1u);
    });
    lds_barrier();
    u64 before;
    const int b = MASS ? crossing(sh.mass, target, before, sh) : crossing(sh.count, target, before, sh);
    target -= before;
    found |= (uint32_t)b << shift;
  }
  if (!MASS)
    above = sum_of(src, sh, [&](int, float l) {
      return bin_of(r, l) == bin && rank_of(l) < found ? fixed(weight(r, l, sh.tab)) : 0;
    });
  return Cut{of_rank(found), target};
}

// The same by the number of the bin's elements (`few` of them): up to 64 are compared with each
// other (`held`: the counts stay), more of a long row are gathered first.
template <bool MASS, class S>
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
    return cut_by_digits<MASS>(r, src, bin, limit, target, above, sh);
  }
  lds_barrier();
  if (t == 0) sh.n = 0;
  lds_barrier();
  each(src, [&](int, float l) {
    if (bin_of(r, l) != bin) return;
    const uint32_t k = rank_of(l);
    if (k >= limit) return;
    const int i = atomicAdd(&sh.n, 1);
    sh.rank[i] = k;
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

// The first whole number that is p times x or more, 1 .. x's own.
__device__ __forceinline__ u64 part_of(float p, u64 x) {
  const double y = (double)p * (double)x;
  u64 n = (u64)y;
  n += (double)n < y;
  return n > 1 ? n : 1;
}

// The cut by top_k (src.n or more: none) and top_p (1 or more: none) among the elements. all_: the
// whole row's sum where the elements are not all that top_p counts, or 0.
template <class S>
__device__ __forceinline__ Cut find_cut(const Row &r, const S &src, int k, float p, u64 all_, Shared &sh) {
  const int t = threadIdx.x;
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
  if (p < 1.0f) block_scan((2 * t < kb ? sh.mass[2 * t] : 0) + (2 * t + 1 < kb ? sh.mass[2 * t + 1] : 0), m_bins, sh);
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

// The first kept element from `start` on at which the running sum passes u times the
// sum, or `goal` where `whole` is given (the sum of a row of which src is a part): the
// range is cut into 16 parts by sums of its waves until it has an element per thread.
// Returns its weight and the sum; -1 where all weights are 0.
template <class S>
__device__ __forceinline__ int draw(const Row &r, const S &src, const Cut &cut, int start, int len, u64 goal, u64 whole,
                                    u64 &w, u64 &sum, Shared &sh) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  auto kept = [&](float l) -> u64 {
    const double x = weight(r, l, sh.tab);
    return x >= r.min_w ? fixed(x) : 0;
  };
  const u64 w_tie = kept(cut.v);
  u64 ties = cut.ties;
  bool first = true;
  auto begin = [&](u64 total) {
    sum = whole ? whole : total;
    if (!whole) goal = (u64)((double)r.u * (double)sum);
    goal = goal < total ? goal : total - 1;  // (a part's sum, as the row's was formed, may be some units off)
    first = false;
  };
  while (len > kThreads) {
    const int part = (len + kThreads - 1) / kThreads * 64, a = start + wave * part;
    const int b = a + part < start + len ? a + part : start + len;
    u64 s = 0;
    uint32_t c = 0;
    constexpr int U = 8;
    int i = a + lane;
    auto add = [&](float l) {
      const u64 x = kept(l);
      s += l > cut.v ? x : 0;
      c += l == cut.v;
    };
    for (; i + (U - 1) * 64 < b; i += U * 64) {
      float x[U];
#pragma unroll
      for (int j = 0; j < U; ++j) x[j] = src.at(i + j * 64);
#pragma unroll
      for (int j = 0; j < U; ++j) add(x[j]);
    }
    for (; i < b; i += 64) add(src.at(i));
    s = wave_scan(s);
    c = (uint32_t)group_sum_i<64>((int)c);
    lds_barrier();
    if (lane == 63) {
      sh.red[wave] = s;
      sh.redi[wave] = c;
    }
    lds_barrier();
    auto of_part = [&](int i, u64 left) { return sh.red[i] + (sh.redi[i] < left ? sh.redi[i] : left) * w_tie; };
    if (first) {
      u64 left = ties, total = 0;
      for (int i = 0; i < kWaves; ++i) {
        total += of_part(i, left);
        left -= sh.redi[i] < left ? sh.redi[i] : left;
      }
      if (!total) return -1;
      begin(total);
    }
    int k = 0;
    for (; k < kWaves - 1; ++k) {
      const u64 m = of_part(k, ties);
      if (goal < m) break;
      goal -= m;
      ties -= sh.redi[k] < ties ? sh.redi[k] : ties;
    }
    const int end = start + len;
    start += k * part;
    len = start + part < end ? part : end - start;
  }
  const float l = t < len ? src.at(start + t) : -INFINITY;
  const bool tie = t < len && l == cut.v;
  u64 total, nth = 0;
  if (ties < kThreads) nth = block_scan(tie, total, sh);
  const u64 m = t < len && (l > cut.v || (tie && nth < ties)) ? kept(l) : 0;
  const u64 x = block_scan(m, total, sh);
  if (first) {
    if (!total) return -1;
    begin(total);
  }
  if (x <= goal && goal < x + m) {
    sh.at = start + t;
    sh.before = m;
  }
  lds_barrier();
  w = sh.before;
  return sh.at;
}

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

typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

// Per chunk of kChunk logits, the largest, the sum of the weights by that one (kFix
// units) where it is asked for, and the largest of every kGroup.
__global__ void __launch_bounds__(256) k_sample_stats(SampleArgs a, int64_t row0, SampleStats st) {
  __shared__ double tab[kTab];
  __shared__ float red[12];
  __shared__ u64 redu[4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = blockIdx.x;
  const int64_t row = row0 + blockIdx.y;
  const float *l = a.logits + row * a.stride;
  const int n = (int)a.n, base = c * kChunk;
  const Settings s(a, row);
  const bool sums = s.sums(a);
  if (sums) make_table(tab);
  float x[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = base + j * 1024 + 4 * t;
    if (i + 4 <= n) {
      const f32x4a4 y = *(const f32x4a4 *)(l + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = clean(y[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = i + e < n ? clean(l[i + e]) : -INFINITY;
    }
  }
  float *gm = st.group_max + ((int64_t)blockIdx.y * gridDim.x + c) * (kChunk / kGroup);
  auto finite = [](float y) { return y == -INFINITY ? INFINITY : y; };  // (-inf is none of the lowest)
  float m = -INFINITY, low = INFINITY, least = INFINITY;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    least = fminf(least, fminf(fminf(finite(x[j][0]), finite(x[j][1])), fminf(finite(x[j][2]), finite(x[j][3]))));
    const float g = group_max<16>(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])));
    if ((lane & 15) == 0) gm[j * 16 + (t >> 4)] = g;
    m = fmaxf(m, g);
    low = fminf(low, finite(g));
  }
  m = group_max<64>(m);
  low = -group_max<64>(-low);
  least = -group_max<64>(-least);
  if (lane == 0) {
    red[wave] = m;
    red[4 + wave] = low;
    red[8 + wave] = least;
  }
  lds_barrier();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  low = fminf(fminf(red[4], red[5]), fminf(red[6], red[7]));
  least = fminf(fminf(red[8], red[9]), fminf(red[10], red[11]));
  u64 sum = 0;
  if (sums) {
    const Row r = s.row(m, 0.0f);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += fixed(weight(r, x[j][e], tab));  // (-inf, past the row's end, weighs nothing)
    sum = wave_scan(sum);
    if (lane == 63) redu[wave] = sum;
    lds_barrier();
    sum = redu[0] + redu[1] + redu[2] + redu[3];
  }
  if (t == 0) {
    st.chunk_max[(int64_t)blockIdx.y * gridDim.x + c] = m;
    st.chunk_low[(int64_t)blockIdx.y * gridDim.x + c] = low;
    st.chunk_min[(int64_t)blockIdx.y * gridDim.x + c] = least;
    st.chunk_sum[(int64_t)blockIdx.y * gridDim.x + c] = sum;
  }
}

// The first element of [start, end) that is l.
__device__ __forceinline__ int first_equal(const Logits &src, int start, int end, float l, Shared &sh) {
  lds_barrier();
  if (threadIdx.x == 0) sh.at = end;
  lds_barrier();
  int first = end;
  for (int i = start + threadIdx.x; i < end && first == end; i += kThreads) first = src.at(i) == l ? i : end;
  if (first < end) atomicMin(&sh.at, first);
  lds_barrier();
  return sh.at;
}

// The elements whose even bin is at most b0, in sh.cand and sh.index, in their order;
// -1 where they are too many. A group's largest says whether it has any.
__device__ __forceinline__ int gather(const Row &r, const Logits &src, const float *gm, int n_group, int b0, Shared &sh) {
  const int t = threadIdx.x, l16 = t & 15;
  int n = 0;
  for (int g0 = 0; g0 < n_group; g0 += kThreads) {
    const int g = g0 + t;
    const float x = g < n_group ? gm[g] : -INFINITY;
    const bool in = x != -INFINITY && bin_of(r, x) <= b0;
    u64 total;
    const int at = n + (int)block_scan(in, total, sh);
    if (in && at < kGroups) sh.group[at] = (uint16_t)g;
    n += (int)total;
  }
  if (n > kGroups) return -1;
  lds_barrier();
  float x[4];  // of the last group that was looked at
  auto load = [&](int i) {
    const int at = sh.group[i] * kGroup + 4 * l16;
    uint32_t in = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = at + e < src.n ? src.at(at + e) : -INFINITY;
      if (x[e] != -INFINITY && bin_of(r, x[e]) <= b0) in |= 1u << e;
    }
    return in;
  };
  uint32_t in = 0;
  for (int i = t >> 4; i < n; i += kThreads / 16) {
    in = load(i);
    const int m = group_sum_i<16>(__builtin_popcount(in));
    if (l16 == 0) sh.in_group[i] = (uint16_t)m;
  }
  lds_barrier();
  u64 total;
  const uint32_t mine = t < n ? sh.in_group[t] : 0;
  const int at = (int)block_scan(mine, total, sh);
  if (total > kCand) return -1;
  if (t < n) sh.in_group[t] = (uint16_t)at;
  lds_barrier();
  for (int i = t >> 4; i < n; i += kThreads / 16) {
    if (n > kThreads / 16) in = load(i);
    int before = __builtin_popcount(in);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      const int y = __shfl_up(before, d, 16);
      if (l16 >= d) before += y;
    }
    int to = sh.in_group[i] + before - __builtin_popcount(in);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (in & (1u << e)) {
        sh.cand[to] = x[e];
        sh.index[to++] = sh.group[i] * kGroup + 4 * l16 + e;
      }
  }
  lds_barrier();
  return (int)total;
}

// A row of which more is kept than fits the candidates, without top_k: `parts` work-groups
// share it. Each sums the weights of its part by bins; the last to arrive finds the cut
// among the elements of the bin that the target falls into, and by the parts' sums the
// part that the drawn token is in, so that only that one is gone through. Returns the token, -1 where
// another work-group ends the row.
__device__ __forceinline__ int draw_flat(const Row &r, const Logits &src, float p, const SampleStats &st, int parts, u64 &w,
                                         u64 &sum, Shared &sh) {
  const int t = threadIdx.x, len = (src.n + parts - 1) / parts, mine = blockIdx.y;
  auto part = [&](int i) {
    const int a = i * len < src.n ? i * len : src.n;
    return Logits{src.l + a, src.n - a < len ? src.n - a : len};
  };
  lds_barrier();
  clear(sh.mass);
  lds_barrier();
  each(part(mine), [&](int, float l) {
    const u64 x = fixed(weight(r, l, sh.tab));
    if (x) atomicAdd(&sh.mass[bin_of(r, l)], x);
  });
  lds_barrier();
  u64 *all = st.part_sum + (int64_t)blockIdx.x * parts * kBins;
  if (parts > 1) {
    // (agent-scope accesses go past the XCDs' caches, and each wave has waited for its
    // stores before the counter's add: no release besides)
    for (int i = t; i < kBins; i += kThreads)
      __hip_atomic_store(all + mine * kBins + i, sh.mass[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0) sh.n = (int)__hip_atomic_fetch_add(st.counters + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (sh.n != parts - 1) return -1;
    if (t == 0) __hip_atomic_store(st.counters + blockIdx.x, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int i = t; i < kBins; i += kThreads) {
      u64 x[kParts], s = 0;
#pragma unroll
      for (int k = 0; k < kParts; ++k)
        x[k] = k < parts ? __hip_atomic_load(all + k * kBins + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
#pragma unroll
      for (int k = 0; k < kParts; ++k) s += x[k];
      sh.mass[i] = s;
    }
    lds_barrier();
  }
  u64 total, before;
  block_scan(sh.mass[2 * t] + sh.mass[2 * t + 1], total, sh);
  u64 target = part_of(p, total);
  target = target < total ? target : total;
  const int b = crossing(sh.mass, target, before, sh);
  // the bin's elements, with their places
  if (t == 0) sh.n = 0;
  lds_barrier();
  each(src, [&](int i, float l) {
    if (bin_of(r, l) != b) return;
    const int k = atomicAdd(&sh.n, 1);
    if (k < kCand) {
      sh.cand[k] = l;
      sh.index[k] = i;
    }
  });
  lds_barrier();
  const int n = sh.n;
  u64 none;
  bool held = true;
  Cut cut;
  if (n > kCand) {
    cut = cut_by_digits<true>(r, src, b, 0xffffffffu, target - before, none, sh);
  } else {
    const Candidates in{sh.cand, n};
    cut = cut_in_bin<true>(r, in, b, n, 0xffffffffu, target - before, none, held, sh);
  }
  const double wt = weight(r, cut.v, sh.tab);
  const u64 w_tie = fixed(wt);
  cut.ties = (cut.ties + w_tie - 1) / w_tie;
  // the parts' sums, where all of the kept weigh min_p and none of the equal ones is left out
  u64 equal = 0;
  if (n <= kCand && parts > 1) {
    if (t < parts) sh.part[t] = 0;
    lds_barrier();
    uint32_t c = 0;
    for (int i = t; i < n; i += kThreads) {
      const float l = sh.cand[i];
      c += l == cut.v;
      if (l >= cut.v) atomicAdd(&sh.part[sh.index[i] / len], fixed(weight(r, l, sh.tab)));
    }
    block_scan(c, equal, sh);
  }
  if (n > kCand || parts == 1 || wt < r.min_w || equal > cut.ties) return draw(r, src, cut, 0, src.n, 0, 0, w, sum, sh);
  for (int k = 0; k < parts; ++k) {
    u64 s = 0, m;
    for (int i = t; i < b; i += kThreads) s += __hip_atomic_load(all + k * kBins + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    block_scan(s, m, sh);
    if (t == 0) sh.part[k] += m;
  }
  lds_barrier();
  sum = 0;
  for (int k = 0; k < parts; ++k) sum += sh.part[k];
  u64 goal = (u64)((double)r.u * (double)sum);
  goal = goal < sum ? goal : sum - 1;
  int k = 0;
  for (; k < parts - 1 && goal >= sh.part[k]; ++k) goal -= sh.part[k];
  const Logits in = part(k);
  lds_barrier();
  return k * len + draw(r, in, Cut{cut.v, ~0ull}, 0, in.n, goal, sum, w, sum, sh);
}

// chunks: 0 without k_sample_stats before it. Grid: (rows, work-groups that share one).
__global__ void __launch_bounds__(kThreads, 1) k_sample(SampleArgs a, int64_t row0, SampleStats st, int chunks) {
  __shared__ Shared sh;
  const int t = threadIdx.x;
  const int64_t row = row0 + blockIdx.x;
  const Settings s(a, row);
  const bool flat = !s.greedy && s.k >= (int)a.n && s.p < 1.0f;  // (the others are one work-group's)
  if (blockIdx.y && !flat) return;
  make_table(sh.tab);
  const Logits src{a.logits + row * a.stride, (int)a.n};
  const float *cm = st.chunk_max + (int64_t)blockIdx.x * chunks;
  // the largest logit, the least and the lowest of the groups' largest (without groups: the least again)
  float m = -INFINITY, least = INFINITY, low = INFINITY;
  if (chunks) {
    const int64_t at = (int64_t)blockIdx.x * chunks;
    for (int i = t; i < chunks; i += kThreads) {
      m = fmaxf(m, cm[i]);
      least = fminf(least, st.chunk_min[at + i]);
      low = fminf(low, st.chunk_low[at + i]);
    }
  } else {
    each(src, [&](int, float l) {
      m = fmaxf(m, l);
      least = fminf(least, l == -INFINITY ? INFINITY : l);
    });
  }
  m = group_max<64>(m);
  least = -group_max<64>(-least);
  low = -group_max<64>(-low);
  if ((t & 63) == 0) {
    sh.redf[0][t >> 6] = m;
    sh.redf[1][t >> 6] = least;
    sh.redf[2][t >> 6] = low;
  }
  lds_barrier();
  for (int i = 0; i < kWaves; ++i) {
    m = fmaxf(m, sh.redf[0][i]);
    least = fminf(least, sh.redf[1][i]);
    low = fminf(low, sh.redf[2][i]);
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
      if (t < chunks && cm[t] == m) atomicMin(&sh.at, t);
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
      if (t < chunks)
        mine = (u64)__builtin_rint((double)st.chunk_sum[(int64_t)blockIdx.x * chunks + t] * 0x1p-43 * weight(r, cm[t], sh.tab));
      before = block_scan(mine, sum, sh);
    }
    int at = -1;
    if (sum && s.p >= 1.0f) {  // everything is kept: the chunk, then the token in it
      u64 goal = (u64)((double)r.u * (double)sum);
      goal = goal < sum ? goal : sum - 1;
      if (before <= goal && goal < before + mine) {
        sh.at = t;
        sh.before = before;
      }
      lds_barrier();
      const int start = sh.at * kChunk, end = start + kChunk < src.n ? start + kChunk : src.n;
      goal -= sh.before;
      const float top = cm[sh.at];
      lds_barrier();
      at = draw(r, src, Cut{-INFINITY, ~0ull}, start, end - start, goal, sum, w, sum, sh);
      id = at >= 0 ? at : first_equal(src, start, end, top, sh);  // (a chunk of many weights of under half a unit)
      w = at >= 0 ? w : 1;
      at = 0;
    } else if (chunks) {
      // a bin that holds the last kept token, or one after it, by the groups' largest: as
      // many of them as tokens are kept, or of as much weight
      const float *gm = st.group_max + (int64_t)blockIdx.x * chunks * (kChunk / kGroup);
      const int n_group = (src.n + kGroup - 1) / kGroup;
      int b0 = kBins;
      lds_barrier();
      if (s.k < src.n) clear(sh.count);
      else clear(sh.mass);
      lds_barrier();
      for (int g = t; g < n_group; g += kThreads) {
        const float x = gm[g];
        if (x == -INFINITY) continue;
        const int b = bin_of(r, x);
        if (s.k < src.n) atomicAdd(&sh.count[b], 1u);
        else if (s.p < 1.0f) atomicAdd(&sh.mass[b], fixed(weight(r, x, sh.tab)));
      }
      lds_barrier();
      u64 total, none;
      if (s.k < src.n) {
        block_scan((u64)sh.count[2 * t] + sh.count[2 * t + 1], total, sh);
        if ((u64)s.k <= total) b0 = crossing(sh.count, (u64)s.k, none, sh);
      } else if (s.p < 1.0f) {
        const u64 target = part_of(s.p, sum);
        block_scan(sh.mass[2 * t] + sh.mass[2 * t + 1], total, sh);
        if (target <= total) b0 = crossing(sh.mass, target, none, sh);
      }
      if (s.min_p > 0.0f && (s.k >= src.n || s.p >= 1.0f)) {
        // (where top_p counts among the top_k all of those are needed)
        const float x = (float)(-log((double)s.min_p) * (double)s.temp) * r.scale + 1.0f;
        b0 = x < (float)b0 ? (int)x : b0;
      }
      if (b0 < kBins - 1) {
        const int n = gather(r, src, gm, n_group, b0, sh);
        if (n >= 0) {
          if (blockIdx.y) return;
          const Candidates cand{sh.cand, n};
          Row f = r;
          f.scale = r.scale * ((float)kBins / (float)(b0 + 1));  // (their bins, finer)
          const Cut cut = find_cut(f, cand, s.k, s.p, s.k < src.n ? 0 : sum, sh);
          at = draw(f, cand, cut, 0, n, 0, 0, w, sum, sh);
          id = sh.index[at];
        }
      }
    }
    if (at < 0) {
      r.scale = s.scale(m, least, flat);
      if (flat) {
        id = draw_flat(r, src, s.p, st, (int)gridDim.y, w, sum, sh);
        if (id < 0) return;
      } else {
        const Cut cut = find_cut(r, src, s.k, s.p, 0, sh);
        id = draw(r, src, cut, 0, src.n, 0, 0, w, sum, sh);
      }
    }
    prob = (float)((double)w / (double)sum);
  }
  if (t == 0) {
    a.out[row] = (uint32_t)id;
    if (a.prob) a.prob[row] = prob;
    if (a.pos) a.pos[row] += a.advance;
  }
}

constexpr int64_t kFewTokens = 8192;  // a work-group reads so many as quickly as another launch comes
constexpr int kShareRows = 256;       // rows times the work-groups that share one

}  // namespace

constexpr size_t kStatBytes = (size_t)16 << 20;
size_t sample_ws_bytes() { return kStatBytes + (size_t)kShareRows * kBins * 8; }
int sample_counters() { return kShareRows; }

hipError_t launch_sample(hipStream_t st, const SampleArgs &a, uint8_t *ws, uint32_t *counters) {
  if (a.n <= kFewTokens) {
    KMOE_LAUNCH(k_sample, dim3((unsigned)a.rows), dim3(kThreads), 0, st, a, (int64_t)0, SampleStats{}, 0);
    return hipGetLastError();
  }
  const int chunks = (int)((a.n + kChunk - 1) / kChunk);
  const int64_t each = (int64_t)chunks * (20 + 4 * (kChunk / kGroup)), most = (int64_t)kStatBytes / each;
  for (int64_t row = 0; row < a.rows; row += most) {
    const int64_t n = a.rows - row < most ? a.rows - row : most;
    // the chip's work-groups among few rows
    const int parts = !a.top_p ? 1 : (int)(kShareRows / n < 1 ? 1 : kShareRows / n < kParts ? kShareRows / n : kParts);
    auto at = [&](int64_t bytes) { return (float *)(ws + bytes * most * chunks); };
    const SampleStats s{(unsigned long long *)ws, at(8), at(12), at(16), at(20), (unsigned long long *)(ws + kStatBytes), counters};
    KMOE_LAUNCH(k_sample_stats, dim3((unsigned)chunks, (unsigned)n), dim3(256), 0, st, a, row, s);
    KMOE_LAUNCH(k_sample, dim3((unsigned)n, (unsigned)parts), dim3(kThreads), 0, st, a, row, s, chunks);
  }
  return hipGetLastError();
}

}  // namespace kmoe
