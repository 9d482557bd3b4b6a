// kmoe_paged_select.hip — pages of a long context that a row attends over: bounds of
// the pages' keys, and the choice of the pages by them.
//
// A page's bounds are the least and the largest key of every dim, lo and hi. A query q
// has no score on the page above sum_d max(q_d lo_d, q_d hi_d), and over the heads of
// a kv head's group that is hi . sum max(q, 0) + lo . sum min(q, 0): one product of
// 2 hd elements per page, whatever the number of heads. Pages whose scores lie next to
// each other decide what a row sees, so scores are formed and compared in 64 bits.
//
// The chosen pages of a row and kv head become a page table of their own (its kv head
// of the pages as a cache of one kv head, the row as a sequence of one row), which the
// paged attention reads as any other: all of them are whole but the last, the row's own,
// which ends the sequence.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kmoe_launch.h"
#include "kmoe_device.h"
#include "kmoe_paged.h"

namespace kmoe {
namespace {

typedef unsigned long long u64;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------- bounds

// The i-th of the pages that the batch's rows lie on: sequence and column. Sequence b's
// lie from row_start[b] / page + 2 b on, which is room for them.
__device__ __forceinline__ bool touched(const PagedArgs &a, int i, int &b, int64_t &col) {
  if (!a.row_start) {
    b = i;
    col = ((int64_t)a.seq_len[b] - 1) / a.page;
    return a.seq_len[b] > 0;
  }
  auto at = [&](int x) -> int64_t {
    int64_t r = a.row_start[x];
    r = r < 0 ? 0 : r < a.s_rows ? r : a.s_rows;
    return r / a.page + 2 * x;
  };
  int lo = 0;
  for (int hi = a.n_seq; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (at(mid) <= i) lo = mid;
    else hi = mid;
  }
  b = lo;
  int64_t r0, n;
  paged_rows(a, b, r0, n);
  const int64_t len = a.seq_len[b], first = len - n > 0 ? (len - n) / a.page : 0;
  col = first + (i - at(b));
  return n > 0 && len > 0 && col >= first && col <= (len - 1) / a.page;
}

// min and max over the 16 positions of the lanes that share a group of dims.
__device__ __forceinline__ float min16(float v) { return -group_max<16>(-v); }

// One wave per page, kv head and 32 (Q8_0: 64) dims: its K tiles one by one, every
// lane eight (sixteen) dims of one position of each.
template <int T>
__global__ void __launch_bounds__(256) k_paged_bounds(PagedArgs a, int n_unit, uint16_t *__restrict__ bounds) {
  constexpr int DIMS = T == kPgF16 ? 32 : 64, E = T == kPgF16 ? 8 : 16;
  const int lane = threadIdx.x & 63, kg = lane >> 4, pos = lane & 15;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int nt = a.hd / DIMS;
  if (unit >= (int64_t)n_unit * a.n_kv * nt) return;
  const int i = (int)(unit / (a.n_kv * nt)), g = (int)(unit / nt % a.n_kv), dt = (int)(unit % nt);
  int b;
  int64_t col;
  if (!touched(a, i, b, col)) return;
  const int64_t bb = paged_block_bytes(T, a.page, a.hd);
  const uint8_t *blk = paged_block(a, bb, b, col * a.page, g);
  if (!blk) return;
  const int64_t left = (int64_t)a.seq_len[b] - col * a.page;
  const int n = left < a.page ? (int)left : a.page;  // positions on the page
  float lo[E], hi[E];
#pragma unroll
  for (int e = 0; e < E; ++e) lo[e] = INFINITY, hi[e] = -INFINITY;
#pragma unroll 2
  for (int p0 = 0; p0 < n; p0 += 16) {
    const int p = p0 + pos < n ? p0 + pos : n - 1;  // (past them: the last one again)
    float x[E];
    if constexpr (T == kPgF16) {
      const h8 k = *(const h8 *)(blk + paged_k_off<T>(a.hd, p, dt * 32 + 8 * kg));
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)k[e];
    } else {
      const uint4 k = *(const uint4 *)(blk + paged_k_off<T>(a.hd, p, dt * 64 + 8 * kg));
      const uint32_t w[4] = {k.x, k.y, k.z, k.w};
      const float d0 = (float)*(const _Float16 *)(blk + paged_ks_off(a.page, a.hd, p, 2 * dt));
      const float d1 = (float)*(const _Float16 *)(blk + paged_ks_off(a.page, a.hd, p, 2 * dt + 1));
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = (float)(int8_t)(w[e >> 2] >> (8 * (e & 3))) * (e < 8 ? d0 : d1);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      lo[e] = fminf(lo[e], x[e]);  // (a NaN is passed over)
      hi[e] = fmaxf(hi[e], x[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    lo[e] = min16(lo[e]);
    hi[e] = group_max<16>(hi[e]);
  }
  if (pos != 0) return;
  const int64_t id = (blk - a.pages) / bb;  // page * n_kv + g
  uint16_t *to = bounds + id * 2 * a.hd + dt * DIMS + 8 * kg;
  // Q8_0: a value is eight bits times eleven, rounded here; one past f16's range would be
  // an infinity, which a zero of q makes NaN
  auto half = [](float x) {
    if (T != kPgF16 && fabsf(x) < INFINITY) x = fminf(fmaxf(x, -65504.0f), 65504.0f);
    return (_Float16)x;
  };
#pragma unroll
  for (int u = 0; u < E / 8; ++u) {
    h8 l, h;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      l[e] = half(lo[8 * u + e]);
      h[e] = half(hi[8 * u + e]);
    }
    *(h8 *)(to + 32 * u) = l;
    *(h8 *)(to + a.hd + 32 * u) = h;
  }
}

// ---------------------------------------------------------------- selection

constexpr int kPart = 512;    // pages that a work-group scores
constexpr int kBins = 1024;

// Order of the scores as whole numbers, the best ones smallest; NaN before all.
__device__ __forceinline__ u64 rank_of(double x) {
  const u64 b = (u64)__double_as_longlong(x + 0.0);
  return x != x ? 0 : ~(b ^ ((u64)((int64_t)b >> 63) | 0x8000000000000000ull));
}
constexpr u64 kNoPage = ~0ull;  // (the rank of no score: -inf's is 0xffefff..)

__device__ __forceinline__ double sum_lanes(double x, int width) {
  for (int d = 1; d < width; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

__device__ __forceinline__ int block_scan(int x, int &total, int *red) {  // exclusive, 256 threads
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int in = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(in, d);
    if (lane >= d) in += y;
  }
  __syncthreads();
  if (lane == 63) red[wave] = in;
  __syncthreads();
  int before = in - x;
  total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) before += red[w];
    total += red[w];
  }
  return before;
}

struct Ranks {
  const u64 *p;
  bool local;  // in LDS, or handed over by other work-groups
  __device__ __forceinline__ u64 at(int i) const {
    return local ? p[i] : __hip_atomic_load(p + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
};

// A work-group: kPart pages of one row and kv head; the last one of a row to arrive
// chooses. Grid: (parts, rows by kv heads).
template <int HD>
__global__ void __launch_bounds__(256) k_paged_select(SelectArgs s, int64_t i0) {
  constexpr int LP = HD / 8;  // lanes that share a page
  __shared__ u64 key[kPart];
  __shared__ int count[kBins];
  __shared__ u64 ext[2][4];
  __shared__ int red[4], last, found[2];
  const PagedArgs &a = s.a;
  const int t = threadIdx.x, lane = t & 63;
  const int64_t i = i0 + blockIdx.y, row = i / a.n_kv;
  const int g = (int)(i - row * a.n_kv);
  // the row's sequence and position
  int b = 0;
  int64_t r0, n;
  if (!a.row_start) {
    b = (int)row;
  } else {
    for (int hi = a.n_seq; hi - b > 1;) {
      const int mid = (b + hi) >> 1;
      if (a.row_start[mid] <= row) b = mid;
      else hi = mid;
    }
  }
  paged_rows(a, b, r0, n);
  const bool in = row >= r0 && row < r0 + n;
  if (a.row_start && blockIdx.x == 0 && t == 0) {  // rows that no sequence has lie before the first and behind the last
    int64_t lo, hi, m;
    paged_rows(a, 0, lo, m);
    paged_rows(a, a.n_seq - 1, hi, m);
    hi += m;
    auto clip = [&](int64_t r) { return r < lo * a.n_kv ? lo * a.n_kv : r > hi * a.n_kv ? hi * a.n_kv : r; };
    s.row_start[blockIdx.y] = (int32_t)(clip(i) - i0);
    if (blockIdx.y == gridDim.y - 1) s.row_start[gridDim.y] = (int32_t)(clip(i + 1) - i0);
  }
  const int64_t cap = (int64_t)a.table_cols * a.page, pos = in ? (int64_t)a.seq_len[b] - n + row - r0 : -1;
  const int64_t end = pos + 1 < cap ? pos + 1 : cap;
  int32_t *to = s.table + (int64_t)blockIdx.y * s.n_select;
  if (end <= 0) {
    if (blockIdx.x == 0 && t == 0) s.len[blockIdx.y] = 0;
    return;
  }
  const int mine = (int)((end - 1) / a.page);  // the row's own column
  const int parts = mine / kPart + 1;
  if ((int)blockIdx.x >= parts) return;
  const int c0 = blockIdx.x * kPart, c1 = c0 + kPart < mine ? c0 + kPart : mine;  // to score: columns before its own
  const int32_t *tab = a.table + (int64_t)b * a.table_cols;
  auto page = [&](int c) {
    const int32_t id = tab[c];
    return id >= 0 && id < a.n_pages ? id : -1;
  };
  const int own = page(mine) >= 0, first = s.n_first < mine ? s.n_first : mine;
  // its heads' positive and negative parts, summed
  const int l = lane % LP;
  double qp[8], qn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) qp[e] = qn[e] = 0.0;
  const float *q = s.q + (row * s.n_head + (int64_t)g * s.group) * HD + 8 * l;
  for (int h = 0; h < s.group; ++h) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double x = q[(int64_t)h * HD + e];
      qp[e] += x > 0.0 ? x : x != x ? x : 0.0;
      qn[e] += x < 0.0 ? x : 0.0;
    }
  }
  for (int c = c0 + t / LP; c < c0 + kPart; c += 256 / LP) {
    u64 k = kNoPage;
    if (c < c1) {  // (uniform among the lanes of a page)
      const int id = page(c);
      if (id >= 0) {
        const uint16_t *bd = s.bounds + ((int64_t)id * a.n_kv + g) * 2 * HD + 8 * l;
        const h8 lo = *(const h8 *)bd, hi = *(const h8 *)(bd + HD);
        double x = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) x = fma((double)(float)lo[e], qn[e], fma((double)(float)hi[e], qp[e], x));
        k = c < first ? 0 : rank_of(sum_lanes(x, LP));
      }
    }
    if (l == 0) key[c - c0] = k;
  }
  __syncthreads();
  Ranks r{key, true};
  if (parts > 1) {
    u64 *all = s.scores + (int64_t)blockIdx.y * a.table_cols;
    for (int c = c0 + t; c < c1; c += 256) __hip_atomic_store(all + c, key[c - c0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0) last = __hip_atomic_fetch_add(s.counters + blockIdx.y, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)parts - 1;
    __syncthreads();
    if (!last) return;
    if (t == 0) __hip_atomic_store(s.counters + blockIdx.y, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    r = Ranks{all, false};
  }
  // The best `want` of the columns before its own. Among those whose rank lies in [lo,
  // hi], the bin of the want-th is found by steps of a power of two, and taken as the
  // next range: ten bits a time, of 64 at most.
  int want = s.n_select - own, have = 0;
  for (int c = t; c < mine; c += 256) have += r.at(c) != kNoPage;
  int total;
  block_scan(have, total, red);
  u64 cut = kNoPage - 1;  // ranks up to it are taken, of those equal to it `ties`
  int ties = INT32_MAX;
  if (want <= 0) {  // its own page alone
    cut = 0;
    ties = 0;
  } else if (total > want) {
    u64 lo = 0, hi = kNoPage - 1;
    for (;;) {
      u64 mn = kNoPage, mx = 0;
      for (int c = t; c < mine; c += 256) {
        const u64 k = r.at(c);
        if (k < lo || k > hi) continue;
        mn = k < mn ? k : mn;
        mx = k > mx ? k : mx;
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const u64 y = __shfl_xor(mn, d), z = __shfl_xor(mx, d);
        mn = y < mn ? y : mn;
        mx = z > mx ? z : mx;
      }
      __syncthreads();
      if (lane == 0) {
        ext[0][t >> 6] = mn;
        ext[1][t >> 6] = mx;
      }
      for (int c = t; c < kBins; c += 256) count[c] = 0;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        mn = ext[0][w] < mn ? ext[0][w] : mn;
        mx = ext[1][w] > mx ? ext[1][w] : mx;
      }
      if (mn == mx) {  // equal ones: the first by column
        cut = mn;
        ties = want;
        break;
      }
      const int shift = 64 - __clzll((long long)(mx - mn)) > 10 ? 64 - __clzll((long long)(mx - mn)) - 10 : 0;
      for (int c = t; c < mine; c += 256) {
        const u64 k = r.at(c);
        if (k >= mn && k <= mx) atomicAdd(&count[(k - mn) >> shift], 1);
      }
      __syncthreads();
      int x[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += x[e] = count[4 * t + e];
      int before = block_scan(sum, total, red);
      if (before < want && before + sum >= want) {
        int e = 0;
        for (; before + x[e] < want; ++e) before += x[e];
        found[0] = 4 * t + e;
        found[1] = before;
      }
      __syncthreads();
      lo = mn + ((u64)found[0] << shift);
      hi = mx - lo > (1ull << shift) - 1 ? lo + ((1ull << shift) - 1) : mx;
      want -= found[1];
      if (shift == 0) {
        cut = lo;
        ties = want;
        break;
      }
    }
  }
  // the chosen ones in the order of their columns, then its own
  int at = 0;
  for (int c = 0; c < mine; c += 256) {
    const u64 k = c + t < mine ? r.at(c + t) : kNoPage;
    int nt = 0, m, before = 0;
    const bool tie = k == cut;
    if (ties != INT32_MAX) before = block_scan(tie, nt, red);
    const bool take = k < cut || (tie && before < ties);
    const int x = at + block_scan(take, m, red);
    if (take) to[x] = tab[c + t] * a.n_kv + g;
    at += m;
    ties = ties == INT32_MAX ? ties : ties - nt;
  }
  if (t == 0) {
    if (own) to[at] = tab[mine] * a.n_kv + g;
    s.len[blockIdx.y] = (int32_t)(at * (int64_t)a.page + (own ? end - (int64_t)mine * a.page : 0));
  }
}

constexpr int64_t kRowsAtOnce = 1024;             // rows by kv heads of a launch
constexpr int64_t kScores = (int64_t)1 << 22;     // of a launch
constexpr int64_t kChosen = (int64_t)1 << 22;

}  // namespace

int64_t select_max_cols() { return (int64_t)1 << 20; }
int select_counters() { return (int)kRowsAtOnce; }
size_t select_ws_bytes() { return kScores * 8 + kChosen * 4 + (2 * kRowsAtOnce + 1) * 4; }

hipError_t launch_paged_bounds(hipStream_t st, const PagedArgs &a, uint16_t *bounds) {
  const int64_t n = a.row_start ? a.s_rows / a.page + 2 * (int64_t)a.n_seq : a.n_seq;
  const int64_t waves = n * a.n_kv * (a.hd / (a.type == kPgF16 ? 32 : 64));
  const dim3 grid((unsigned)((waves + 3) / 4));
  if (a.type == kPgF16) KMOE_LAUNCH(k_paged_bounds<kPgF16>, grid, dim3(256), 0, st, a, (int)n, bounds);
  else KMOE_LAUNCH(k_paged_bounds<kPgQ8>, grid, dim3(256), 0, st, a, (int)n, bounds);
  return hipGetLastError();
}

hipError_t launch_paged_attention_selected(hipStream_t st, const PagedArgs &a, const uint16_t *bounds, const float *q,
                                           int n_head, int n_select, int n_first, float *out, float *part,
                                           uint32_t *counters, uint8_t *ws, uint32_t *select_counters) {
  const int group = n_head / a.n_kv, n_sel = n_select < a.table_cols ? n_select : a.table_cols;
  const int64_t units = a.s_rows * a.n_kv;
  const int64_t most = std::min(std::min(kRowsAtOnce, kScores / a.table_cols), kChosen / n_sel);
  SelectArgs s{a, bounds, q, n_head, group, n_sel, n_first, (unsigned long long *)ws, (int32_t *)(ws + kScores * 8), nullptr, nullptr, select_counters};
  s.len = s.table + kChosen;
  s.row_start = s.len + kRowsAtOnce;
  for (int64_t i = 0; i < units; i += most) {
    const int n = (int)std::min(most, units - i);
    const dim3 grid((unsigned)((a.table_cols + kPart - 1) / kPart), (unsigned)n);
    if (a.hd == 64) KMOE_LAUNCH(k_paged_select<64>, grid, dim3(256), 0, st, s, i);
    else KMOE_LAUNCH(k_paged_select<128>, grid, dim3(256), 0, st, s, i);
    PagedArgs p = a;
    p.n_kv = 1;
    p.n_pages = a.n_pages * a.n_kv;
    p.n_seq = n;
    p.table_cols = n_sel;
    p.s_rows = n;
    p.row_start = a.row_start ? s.row_start : nullptr;
    p.seq_len = s.len;
    p.table = s.table;
    const int64_t at = i * group * a.hd;
    const hipError_t e = launch_paged_attention(st, p, q + at, group, 0, 0, out + at, part, counters);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace kmoe
