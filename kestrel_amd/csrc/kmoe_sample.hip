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
  const float *l;
  int n;
  float max;     // largest logit
  double inv_t;  // 1 / T
  float scale;   // bins per unit of logit
  int k;         // tokens kept at most
  float p;       // >= 1: all
  double min_p;  // 0: all
  float u;
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
  u64 before;
  int at;
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

// f(i, l) for every element i of the row, a work-group together.
template <class F>
__device__ __forceinline__ void each(const Row &r, F &&f) {
  constexpr int U = 8;
  int i = threadIdx.x;
  for (; i + (U - 1) * kThreads < r.n; i += U * kThreads) {
    float x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) x[j] = r.l[i + j * kThreads];
#pragma unroll
    for (int j = 0; j < U; ++j) f(i + j * kThreads, clean(x[j]));
  }
  for (; i < r.n; i += kThreads) f(i, clean(r.l[i]));
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
template <bool MASS>
__device__ Cut cut_in_bin(const Row &r, int bin, uint32_t limit, u64 target, Shared &sh) {
  uint32_t found = 0;
#pragma unroll 1
  for (int d = 0; d < 3; ++d) {  // 11, 11 and 10 bits
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, top = d == 0 ? 32 : d == 1 ? 21 : 10;
    __syncthreads();
    if (MASS) clear(sh.mass);
    else clear(sh.count);
    __syncthreads();
    each(r, [&](int, float l) {
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

// Sum of f(i, l) over the row, to every thread.
template <class F>
__device__ __forceinline__ u64 sum_of(const Row &r, Shared &sh, F &&f) {
  u64 s = 0, total;
  each(r, [&](int i, float l) { s += f(i, l); });
  block_scan(s, total, sh);
  return total;
}

// The first kept token, by index, at which the running sum passes u times the whole:
// the range is cut into 16 parts by sums of its waves until it has an element per thread.
// Returns its weight and the sum.
__device__ int draw(const Row &r, const Cut &cut, u64 &w, u64 &sum, Shared &sh) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  auto kept = [&](float l) -> u64 {
    const double x = weight(r, l, sh.tab);
    return x >= r.min_p ? fixed(x) : 0;
  };
  const u64 w_tie = kept(of_rank(cut.rank));
  int start = 0, len = r.n;
  u64 goal = 0, ties = cut.ties;
  bool first = true;
  while (len > kThreads) {
    const int part = (len + kThreads - 1) / kThreads * 64, a = start + wave * part;
    const int b = a + part < start + len ? a + part : start + len;
    u64 s = 0;
    uint32_t c = 0;
#pragma unroll 4
    for (int i = a + lane; i < b; i += 64) {
      const float l = clean(r.l[i]);
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
      u64 left = ties;
      sum = 0;
      for (int i = 0; i < kWaves; ++i) {
        sum += of_part(i, left);
        left -= sh.redi[i] < left ? sh.redi[i] : left;
      }
      goal = (u64)((double)r.u * (double)sum);
      goal = goal < sum ? goal : sum - 1;
      first = false;
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
  const float l = t < len ? clean(r.l[start + t]) : 0.0f;
  const uint32_t k = rank_of(l);
  const bool tie = t < len && k == cut.rank;
  u64 total;
  const u64 nth = block_scan(tie, total, sh);
  const u64 m = t < len && (k < cut.rank || (tie && nth < ties)) ? kept(l) : 0;
  const u64 x = block_scan(m, total, sh);
  if (first) {
    sum = total;
    goal = (u64)((double)r.u * (double)sum);
    goal = goal < sum ? goal : sum - 1;
  }
  if (x <= goal && goal < x + m) {
    sh.at = start + t;
    sh.before = m;
  }
  __syncthreads();
  w = sh.before;
  return sh.at;
}

__global__ void __launch_bounds__(kThreads, 1) k_sample(SampleArgs a) {
  __shared__ Shared sh;
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  if (t < 64) sh.tab[t] = exp2((double)t / 64);
  Row r;
  r.l = a.logits + row * a.stride;
  r.n = (int)a.n;
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  r.k = a.top_k ? a.top_k[row] : 0;
  r.k = r.k > 0 && r.k < r.n ? r.k : r.n;
  r.p = a.top_p ? a.top_p[row] : 1.0f;
  r.p = r.p == r.p ? r.p : 1.0f;
  const float mp = a.min_p ? a.min_p[row] : 0.0f;
  r.min_p = mp > 0.0f ? (double)fminf(mp, 1.0f) : 0.0;
  r.u = a.u[row];
  r.u = r.u > 0.0f ? fminf(r.u, 1.0f) : 0.0f;
  // the largest logit
  float m = -INFINITY;
  each(r, [&](int, float l) { m = fmaxf(m, l); });
  m = group_max<64>(m);
  __shared__ float red[kWaves];
  if ((t & 63) == 0) red[t >> 6] = m;
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) m = fmaxf(m, red[i]);
  r.max = m;
  uint32_t id = 0;
  float prob = 0.0f;
  if (m == -INFINITY) {  // nothing to draw from
  } else if (!(temp > 0.0f) || r.k == 1 || r.p <= 0.0f) {
    if (t == 0) sh.at = r.n;
    __syncthreads();
    int first = r.n;
    each(r, [&](int i, float l) { first = l == m && i < first ? i : first; });
    if (first < r.n) atomicMin(&sh.at, first);
    __syncthreads();
    id = (uint32_t)sh.at;
    prob = 1.0f;
  } else {
    r.inv_t = 1.0 / (double)temp;
    r.scale = fminf((float)(kBins / kSpan * r.inv_t), 3.0e38f);
    Cut cut{0xffffffffu, ~0ull};
    if (r.k < r.n || r.p < 1.0f) {
      clear(sh.mass);
      clear(sh.count);
      __syncthreads();
      each(r, [&](int, float l) {
        const int b = bin_of(r, l);
        atomicAdd(&sh.count[b], 1u);
        const u64 w = fixed(weight(r, l, sh.tab));
        if (w) atomicAdd(&sh.mass[b], w);
      });
      __syncthreads();
      // the bins' sums are used up by the digits' later: everything that is needed of
      // them is found first
      u64 n_before = 0, m_bins = 0, total;
      int kb = kBins;
      if (r.k < r.n) {
        kb = crossing(sh.count, (u64)r.k, n_before, sh);
        const u64 x = (2 * t < kb ? sh.mass[2 * t] : 0) + (2 * t + 1 < kb ? sh.mass[2 * t + 1] : 0);
        block_scan(x, m_bins, sh);
      } else {
        block_scan(sh.mass[2 * t] + sh.mass[2 * t + 1], m_bins, sh);
      }
      u64 all = m_bins, w_tie = 0, m_above = m_bins;
      if (kb < kBins) {
        // (the masses are kept: this counts)
        cut = cut_in_bin<false>(r, kb, 0xffffffffu, (u64)r.k - n_before, sh);
        w_tie = fixed(weight(r, of_rank(cut.rank), sh.tab));
        m_above += sum_of(r, sh, [&](int, float l) {
          return bin_of(r, l) == kb && rank_of(l) < cut.rank ? fixed(weight(r, l, sh.tab)) : 0;
        });
        all = m_above + cut.ties * w_tie;
      }
      if (r.p < 1.0f) {
        const double x = (double)r.p * (double)all;
        u64 target = (u64)x;
        target += (double)target < x;
        target = target > 1 ? target : 1;
        target = target < all ? target : all;
        if (target <= m_bins) {
          u64 before;
          const int b = crossing(sh.mass, target, before, sh);
          cut = cut_in_bin<true>(r, b, 0xffffffffu, target - before, sh);
          w_tie = fixed(weight(r, of_rank(cut.rank), sh.tab));
          cut.ties = (cut.ties + w_tie - 1) / w_tie;
        } else if (target <= m_above) {
          cut = cut_in_bin<true>(r, kb, cut.rank, target - m_bins, sh);
          w_tie = fixed(weight(r, of_rank(cut.rank), sh.tab));
          cut.ties = (cut.ties + w_tie - 1) / w_tie;
        } else {
          cut.ties = (target - m_above + w_tie - 1) / w_tie;
        }
      }
    }
    u64 w, sum;
    id = (uint32_t)draw(r, cut, w, sum, sh);
    prob = (float)((double)w / (double)sum);
  }
  if (t == 0) {
    a.out[row] = id;
    if (a.prob) a.prob[row] = prob;
    if (a.pos) a.pos[row] += a.advance;
  }
}

}  // namespace

hipError_t launch_sample(hipStream_t st, const SampleArgs &a) {
  KMOE_LAUNCH(k_sample, dim3((unsigned)a.rows), dim3(kThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace kmoe
