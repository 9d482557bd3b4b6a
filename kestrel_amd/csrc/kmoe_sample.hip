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

#include "kmoe_device.h"
#include "kmoe_launch.h"

namespace kmoe {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kFix = 43;    // weights in units of 2^-43
constexpr int kBins = 2048;
constexpr u64 kOne = 1ull << kFix;
constexpr int kGroup = 64, kChunk = 4096;  // elements of which k_sample_stats finds the largest, and the sum
constexpr int kCand = 2048, kGroups = 1024;
constexpr float kSpan = 24.0f;  // distances from the largest logit that the even bins tell apart, in units of T

// Order of the logits as whole numbers: the larger the logit, the smaller its rank
// (NaN as -inf, -0 as 0).
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return ~(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u));
}
__device__ __forceinline__ float of_rank(uint32_t r) {
  const uint32_t k = ~r;
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// What one row is drawn by.
struct Row {
  float max;     // largest logit
  double inv_t;  // 1 / T
  float scale;   // bins per unit of logit
  double min_p;  // 0: all
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

// exp(x), -31 <= x <= 0: 2^(i / 64) from a table (LDS) times the exponential of what is
// left, at most log(2) / 128, by its series: the sixth power's term is 2^-54.6.
__device__ __forceinline__ double exp_of(double x, const double *tab) {
  const double i = __builtin_rint(x * 92.332482616893656877);  // 64 / log 2
  double r = fma(i, -0x1.62e42fefa3800p-7, x);                // log(2) / 64, its first 42 bits: exact times i
  r = fma(i, -0x1.ef35793c76730p-51, r);
  const int k = (int)i;
  double y = fma(r, 1.0 / 120, 1.0 / 24);
  y = fma(r, y, 1.0 / 6);
  y = fma(r, y, 0.5);
  y = fma(r, y, 1.0);
  y = r * y;
  const double t = tab[k & 63];
  return ldexp(fma(t, y, t), k >> 6);
}
__device__ __forceinline__ double weight(const Row &r, float l, const double *tab) {
  if (l == r.max) return 1.0;
  const double x = ((double)l - (double)r.max) * r.inv_t;
  return x > -31.0 && l != -INFINITY ? exp_of(x, tab) : 0.0;  // (exp(-31) is under half a unit)
}
// To the nearest unit: 2^52 and a number below it have a last bit of 1.
__device__ __forceinline__ u64 fixed(double w) {
  return (u64)__double_as_longlong(w * 0x1p43 + 0x1p52) & ((1ull << 52) - 1);
}

// Even bins by the distance from the largest logit (not descending where the logits descend).
__device__ __forceinline__ int bin_of(const Row &r, float l) {
  if (l == r.max) return 0;
  return (int)fminf((r.max - l) * r.scale, (float)(kBins - 1));
}

struct Shared {
  double tab[64];
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 red[kWaves];
  uint32_t redi[kWaves];
  float redf[kWaves];
  u64 before;
  int at;
  // candidates, and the groups that they are in with how many candidates each has
  float cand[kCand];
  int index[kCand];
  uint16_t group[kGroups], in_group[kGroups];
};

__device__ __forceinline__ u64 shfl_up64(u64 x, int d) {
  const uint32_t lo = __shfl_up((uint32_t)x, d), hi = __shfl_up((uint32_t)(x >> 32), d);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_scan(u64 x) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 y = shfl_up64(x, d);
    if (lane >= d) x += y;
  }
  return x;
}
// Exclusive scan over the work-group's threads, and the total.
__device__ __forceinline__ u64 block_scan(u64 x, u64 &total, Shared &sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 in = wave_scan(x);
  __syncthreads();  // (the last call's sums are read)
  if (lane == 63) sh.red[wave] = in;
  __syncthreads();
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
  __syncthreads();
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

// A beginning of the order: ranks below `rank`, and the first `ties` of those equal to it.
struct Cut {
  uint32_t rank;
  u64 ties;
};

// Where the running sum over the elements of an even bin whose rank is below `limit`
// reaches target (1 .. their sum): the value's rank, and what is left of the target
// there. MASS: sums of weights, otherwise numbers of elements. Digit by digit.
template <bool MASS, class S>
__device__ __forceinline__ Cut cut_in_bin(const Row &r, const S &src, int bin, uint32_t limit, u64 target, Shared &sh) {
  uint32_t found = 0;
#pragma unroll 1
  for (int d = 0; d < 3; ++d) {  // 11, 11 and 10 bits
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, top = d == 0 ? 32 : d == 1 ? 21 : 10;
    __syncthreads();
    if (MASS) clear(sh.mass);
    else clear(sh.count);
    __syncthreads();
    each(src, [&](int, float l) {
      if (bin_of(r, l) != bin) return;
      const uint32_t k = rank_of(l);
      if (k >= limit || (d && k >> top != found >> top)) return;
      const int b = (k >> shift) & (d == 2 ? 1023 : 2047);
      if (MASS) atomicAdd(&sh.mass[b], fixed(weight(r, l, sh.tab)));
      else atomicAdd(&sh.count[b], 1u);
    });
    __syncthreads();
    u64 before;
    const int b = MASS ? crossing(sh.mass, target, before, sh) : crossing(sh.count, target, before, sh);
    target -= before;
    found |= (uint32_t)b << shift;
  }
  return Cut{found, target};
}

// Sum of f(i, l) over the elements, to every thread.
template <class S, class F>
__device__ __forceinline__ u64 sum_of(const S &src, Shared &sh, F &&f) {
  u64 s = 0, total;
  each(src, [&](int i, float l) { s += f(i, l); });
  block_scan(s, total, sh);
  return total;
}

// The cut by top_k (src.n or more: none) and top_p (1 or more: none) among the elements. all_: the
// whole row's sum where the elements are not all that top_p counts, or 0.
template <class S>
__device__ __forceinline__ Cut find_cut(const Row &r, const S &src, int k, float p, u64 all_, Shared &sh) {
  const int t = threadIdx.x;
  Cut cut{0xffffffffu, ~0ull};
  if (k >= src.n && p >= 1.0f) return cut;
  __syncthreads();
  clear(sh.mass);
  clear(sh.count);
  __syncthreads();
  each(src, [&](int, float l) {
    const int b = bin_of(r, l);
    atomicAdd(&sh.count[b], 1u);
    const u64 w = p < 1.0f ? fixed(weight(r, l, sh.tab)) : 0;
    if (w) atomicAdd(&sh.mass[b], w);
  });
  __syncthreads();
  // k falls into bin kb; m_bins: the sum of the bins before it, m_above: of all elements
  // before the k-th's value
  u64 n_before = 0, m_bins = 0, w_tie = 0;
  int kb = kBins;
  if (k < src.n) kb = crossing(sh.count, (u64)k, n_before, sh);
  block_scan((2 * t < kb ? sh.mass[2 * t] : 0) + (2 * t + 1 < kb ? sh.mass[2 * t + 1] : 0), m_bins, sh);
  u64 m_above = m_bins, all = m_bins;
  if (kb < kBins) {
    cut = cut_in_bin<false>(r, src, kb, 0xffffffffu, (u64)k - n_before, sh);  // (the masses stay)
    if (p >= 1.0f) return cut;
    w_tie = fixed(weight(r, of_rank(cut.rank), sh.tab));
    m_above += sum_of(src, sh, [&](int, float l) {
      return bin_of(r, l) == kb && rank_of(l) < cut.rank ? fixed(weight(r, l, sh.tab)) : 0;
    });
    all = m_above + cut.ties * w_tie;
  }
  const u64 whole = all_ ? all_ : all;
  const double x = (double)p * (double)whole;
  u64 target = (u64)x;
  target += (double)target < x;
  target = target > 1 ? target : 1;
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
  uint32_t limit = cut.rank;
  if (target <= m_bins) {
    b = crossing(sh.mass, target, before, sh);
    limit = 0xffffffffu;
  }
  cut = cut_in_bin<true>(r, src, b, limit, target - before, sh);
  w_tie = fixed(weight(r, of_rank(cut.rank), sh.tab));
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
    return x >= r.min_p ? fixed(x) : 0;
  };
  const u64 w_tie = kept(of_rank(cut.rank));
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
#pragma unroll 4
    for (int i = a + lane; i < b; i += 64) {
      const float l = src.at(i);
      const uint32_t k = rank_of(l);
      if (k < cut.rank) s += kept(l);
      c += k == cut.rank;
    }
    s = wave_scan(s);
    c = (uint32_t)group_sum_i<64>((int)c);
    __syncthreads();
    if (lane == 63) {
      sh.red[wave] = s;
      sh.redi[wave] = c;
    }
    __syncthreads();
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
    int i = 0;
    for (; i < kWaves - 1; ++i) {
      const u64 m = of_part(i, ties);
      if (goal < m) break;
      goal -= m;
      ties -= sh.redi[i] < ties ? sh.redi[i] : ties;
    }
    const int end = start + len;
    start += i * part;
    len = start + part < end ? part : end - start;
  }
  const float l = t < len ? src.at(start + t) : 0.0f;
  const uint32_t k = rank_of(l);
  const bool tie = t < len && k == cut.rank;
  u64 total;
  const u64 nth = block_scan(tie, total, sh);
  const u64 m = t < len && (k < cut.rank || (tie && nth < ties)) ? kept(l) : 0;
  const u64 x = block_scan(m, total, sh);
  if (first) {
    if (!total) return -1;
    begin(total);
  }
  if (x <= goal && goal < x + m) {
    sh.at = start + t;
    sh.before = m;
  }
  __syncthreads();
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
  // whether the sum of all weights is asked for
  __device__ __forceinline__ bool sums(const SampleArgs &a) const { return !greedy && k >= (int)a.n && (p < 1.0f || min_p == 0.0f); }
};

typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

// Per chunk of kChunk logits, the largest, the sum of the weights by that one (kFix
// units) where it is asked for, and the largest of every kGroup.
__global__ void __launch_bounds__(256) k_sample_stats(SampleArgs a, int64_t row0, SampleStats st) {
  __shared__ double tab[64];
  __shared__ float red[4];
  __shared__ u64 redu[4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = blockIdx.x;
  const int64_t row = row0 + blockIdx.y;
  const float *l = a.logits + row * a.stride;
  const int n = (int)a.n, base = c * kChunk;
  const Settings s(a, row);
  const bool sums = s.sums(a);
  if (sums && t < 64) tab[t] = exp2((double)t / 64);
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
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float g = group_max<16>(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])));
    if ((lane & 15) == 0) gm[j * 16 + (t >> 4)] = g;
    m = fmaxf(m, g);
  }
  m = group_max<64>(m);
  if (lane == 0) red[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  u64 sum = 0;
  if (sums) {
    Row r;
    r.max = m;
    r.inv_t = 1.0 / (double)s.temp;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (base + j * 1024 + 4 * t + e < n) sum += fixed(weight(r, x[j][e], tab));
    sum = wave_scan(sum);
    if (lane == 63) redu[wave] = sum;
    __syncthreads();
    sum = redu[0] + redu[1] + redu[2] + redu[3];
  }
  if (t == 0) {
    st.chunk_max[(int64_t)blockIdx.y * gridDim.x + c] = m;
    st.chunk_sum[(int64_t)blockIdx.y * gridDim.x + c] = sum;
  }
}

// The first element of [start, end) that is l.
__device__ __forceinline__ int first_equal(const Logits &src, int start, int end, float l, Shared &sh) {
  __syncthreads();
  if (threadIdx.x == 0) sh.at = end;
  __syncthreads();
  int first = end;
  for (int i = start + threadIdx.x; i < end && first == end; i += kThreads) first = src.at(i) == l ? i : end;
  if (first < end) atomicMin(&sh.at, first);
  __syncthreads();
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
  __syncthreads();
  auto load = [&](int i, float (&x)[4]) {
    const int at = sh.group[i] * kGroup + 4 * l16;
    uint32_t in = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = at + e < src.n ? src.at(at + e) : -INFINITY;
      if (x[e] != -INFINITY && bin_of(r, x[e]) <= b0) in |= 1u << e;
    }
    return in;
  };
  for (int i = t >> 4; i < n; i += kThreads / 16) {
    float x[4];
    const int m = group_sum_i<16>(__builtin_popcount(load(i, x)));
    if (l16 == 0) sh.in_group[i] = (uint16_t)m;
  }
  __syncthreads();
  u64 total;
  const uint32_t mine = t < n ? sh.in_group[t] : 0;
  const int at = (int)block_scan(mine, total, sh);
  if (total > kCand) return -1;
  if (t < n) sh.in_group[t] = (uint16_t)at;
  __syncthreads();
  for (int i = t >> 4; i < n; i += kThreads / 16) {
    float x[4];
    const uint32_t in = load(i, x);
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
  __syncthreads();
  return (int)total;
}

// chunks: 0 without k_sample_stats before it.
__global__ void __launch_bounds__(kThreads, 1) k_sample(SampleArgs a, int64_t row0, SampleStats st, int chunks) {
  __shared__ Shared sh;
  const int t = threadIdx.x;
  const int64_t row = row0 + blockIdx.x;
  if (t < 64) sh.tab[t] = exp2((double)t / 64);
  const Logits src{a.logits + row * a.stride, (int)a.n};
  const Settings s(a, row);
  const float *cm = st.chunk_max + (int64_t)blockIdx.x * chunks;
  // the largest logit
  float m = -INFINITY;
  if (chunks) {
    for (int i = t; i < chunks; i += kThreads) m = fmaxf(m, cm[i]);
  } else {
    each(src, [&](int, float l) { m = fmaxf(m, l); });
  }
  m = group_max<64>(m);
  if ((t & 63) == 0) sh.redf[t >> 6] = m;
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) m = fmaxf(m, sh.redf[i]);
  Row r;
  r.max = m;
  r.u = a.u[row];
  r.u = r.u > 0.0f ? fminf(r.u, 1.0f) : 0.0f;
  r.min_p = s.min_p;
  r.inv_t = 1.0 / (double)s.temp;
  r.scale = fminf((float)(kBins / kSpan * r.inv_t), 3.0e38f);
  int id = 0;
  float prob = 0.0f;
  if (m == -INFINITY) {  // nothing to draw from
  } else if (s.greedy) {
    int start = 0, end = src.n;
    if (chunks) {
      if (t == 0) sh.at = chunks;
      __syncthreads();
      if (t < chunks && cm[t] == m) atomicMin(&sh.at, t);
      __syncthreads();
      start = sh.at * kChunk;
      end = start + kChunk < end ? start + kChunk : end;
    }
    id = first_equal(src, start, end, m, sh);
    prob = 1.0f;
  } else {
    // the chunks' sums by the row's largest
    u64 sum = 0, w = 0, mine = 0, before = 0;
    if (chunks && s.sums(a)) {
      if (t < chunks) {
        Row q = r;
        mine = (u64)__builtin_rint((double)st.chunk_sum[(int64_t)blockIdx.x * chunks + t] * weight(q, cm[t], sh.tab));
      }
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
      __syncthreads();
      const int start = sh.at * kChunk, end = start + kChunk < src.n ? start + kChunk : src.n;
      goal -= sh.before;
      const float cl = cm[sh.at];
      __syncthreads();
      at = draw(r, src, Cut{0xffffffffu, ~0ull}, start, end - start, goal, sum, w, sum, sh);
      id = at >= 0 ? at : first_equal(src, start, end, cl, sh);  // (a chunk of many weights of under half a unit)
      w = at >= 0 ? w : 1;
      at = 0;
    } else if (chunks) {
      // a bin that holds the last kept token, or one after it, by the groups' largest: as
      // many of them as tokens are kept, or of as much weight
      const float *gm = st.group_max + (int64_t)blockIdx.x * chunks * (kChunk / kGroup);
      const int n_group = (src.n + kGroup - 1) / kGroup;
      int b0 = kBins;
      clear(sh.mass);
      clear(sh.count);
      __syncthreads();
      for (int g = t; g < n_group; g += kThreads) {
        const float x = gm[g];
        if (x == -INFINITY) continue;
        const int b = bin_of(r, x);
        if (s.k < src.n) atomicAdd(&sh.count[b], 1u);
        else if (s.p < 1.0f) atomicAdd(&sh.mass[b], fixed(weight(r, x, sh.tab)));
      }
      __syncthreads();
      u64 total, none;
      if (s.k < src.n) {
        block_scan((u64)sh.count[2 * t] + sh.count[2 * t + 1], total, sh);
        if ((u64)s.k <= total) b0 = crossing(sh.count, (u64)s.k, none, sh);
      } else if (s.p < 1.0f) {
        const double x = (double)s.p * (double)sum;
        u64 target = (u64)x;
        target += (double)target < x;
        target = target > 1 ? target : 1;
        block_scan(sh.mass[2 * t] + sh.mass[2 * t + 1], total, sh);
        if (target <= total) b0 = crossing(sh.mass, target, none, sh);
      }
      if (r.min_p > 0.0 && (s.k >= src.n || s.p >= 1.0f)) {
        // (where top_p counts among the top_k all of those are needed)
        const float x = (float)(-log(r.min_p) * (double)s.temp) * r.scale + 1.0f;
        b0 = x < (float)b0 ? (int)x : b0;
      }
      if (b0 < kBins - 1) {
        const int n = gather(r, src, gm, n_group, b0, sh);
        if (n >= 0) {
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
      const Cut cut = find_cut(r, src, s.k, s.p, 0, sh);
      id = draw(r, src, cut, 0, src.n, 0, 0, w, sum, sh);
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

}  // namespace

size_t sample_ws_bytes() { return (size_t)16 << 20; }

hipError_t launch_sample(hipStream_t st, const SampleArgs &a, uint8_t *ws) {
  if (a.n <= kFewTokens) {
    KMOE_LAUNCH(k_sample, dim3((unsigned)a.rows), dim3(kThreads), 0, st, a, (int64_t)0, SampleStats{}, 0);
    return hipGetLastError();
  }
  const int chunks = (int)((a.n + kChunk - 1) / kChunk);
  const int64_t each = (int64_t)chunks * (12 + 4 * (kChunk / kGroup)), most = (int64_t)sample_ws_bytes() / each;
  for (int64_t row = 0; row < a.rows; row += most) {
    const int64_t n = a.rows - row < most ? a.rows - row : most;
    const SampleStats s{(unsigned long long *)ws, (float *)(ws + 8 * most * chunks), (float *)(ws + 12 * most * chunks)};
    KMOE_LAUNCH(k_sample_stats, dim3((unsigned)chunks, (unsigned)n), dim3(256), 0, st, a, row, s);
    KMOE_LAUNCH(k_sample, dim3((unsigned)n), dim3(kThreads), 0, st, a, row, s, chunks);
  }
  return hipGetLastError();
}

}  // namespace kmoe
