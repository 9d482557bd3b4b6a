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
#include "kmoe_scan.h"

namespace kmoe {
namespace {

typedef uint64_t u64;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

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
// lane eight (sixteen) dims of one position of each, as the store laid them: 16 contiguous bytes.
// Bound by the launch (64 pages of 8 kv heads 5 us, of which a page's tiles take 1).
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

constexpr int kPart = 512;    // pages that a work-group scores at most
constexpr int kBins = 1024;
constexpr int kHeld = 4096;   // columns whose ranks are chosen among in LDS

// Order of the scores as whole numbers, the best ones smallest; NaN before all.
__device__ __forceinline__ u64 rank_of(double x) {
  const u64 b = (u64)__double_as_longlong(x + 0.0);
  return x != x ? 0 : ~(b ^ ((u64)((int64_t)b >> 63) | 0x8000000000000000ull));
}
constexpr u64 kNoPage = ~0ull;  // (the rank of no score: -inf's is 0xffefff..)

__device__ __forceinline__ int block_scan(int x, int &total, int *red) {  // exclusive, 256 threads
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int in = wave_scan_i(x);
  lds_barrier();
  if (lane == 63) red[wave] = in;
  lds_barrier();
  int before = in - x;
  total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) before += red[w];
    total += red[w];
  }
  return before;
}

// Ranks of a row's columns, in LDS or as other work-groups handed them over.
struct Held {
  const u64 *p;  // (LDS)
  int n;
  __device__ __forceinline__ u64 at(int i) const { return p[i]; }
};
struct Handed {
  const u64 *p;
  int n;
  __device__ __forceinline__ u64 at(int i) const { return __hip_atomic_load(p + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
};
// f(c, rank) for all of them, a work-group together, eight a thread on their way at a time.
template <class R, class F>
__device__ __forceinline__ void each(const R &r, F &&f) {
  constexpr int U = 8;
  for (int c = threadIdx.x; c < r.n; c += 256 * U) {
    u64 k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = r.at(c + 256 * u < r.n ? c + 256 * u : c);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + 256 * u < r.n) f(c + 256 * u, k[u]);
  }
}

struct Choice {
  u64 ext[2][4], few[64];
  int count[kBins], red[4], found[2], n_few;
};

// The best `want` of the columns, into `to` in their order; how many there are. Among those
// whose rank lies in [lo, hi], the bin of the want-th is found by steps of a power of
// two, and taken as the next range: ten bits a time, of 64 at most, until it holds few.
template <class R>
__device__ __forceinline__ int choose(const R &r, int want, const int32_t *tab, int n_kv, int g, int32_t *to, Choice &sh) {
  const int t = threadIdx.x, lane = t & 63;
  int have = 0, total;
  u64 lo = 0, hi = kNoPage - 1;
  u64 cut = kNoPage - 1;  // ranks up to it are taken, of those equal to it `ties`
  int ties = INT32_MAX;
  for (bool begun = false;; begun = true) {
    u64 mn = kNoPage, mx = 0;
    each(r, [&](int, u64 k) {
      have += k != kNoPage;
      const bool in = k >= lo && k <= hi;
      mn = in && k < mn ? k : mn;
      mx = in && k > mx ? k : mx;
    });
    wave_range(mn, mx);
    if (!begun) {
      block_scan(have, total, sh.red);
      if (total <= want) break;  // all of them
      if (want <= 0) return 0;
    }
    lds_barrier();
    if (lane == 63) {
      sh.ext[0][t >> 6] = mn;
      sh.ext[1][t >> 6] = mx;
    }
#pragma unroll
    for (int e = 0; e < kBins / 256; ++e) sh.count[256 * e + t] = 0;
    if (t == 0) sh.n_few = 0;
    lds_barrier();
    mn = sh.ext[0][0];
    mx = sh.ext[1][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      mn = sh.ext[0][w] < mn ? sh.ext[0][w] : mn;
      mx = sh.ext[1][w] > mx ? sh.ext[1][w] : mx;
    }
    if (mn == mx) {  // equal ones: the first by column
      cut = mn;
      ties = want;
      break;
    }
    const int bits = 64 - __clzll((long long)(mx - mn)), shift = bits > 10 ? bits - 10 : 0;
    each(r, [&](int, u64 k) {
      if (k >= mn && k <= mx) atomicAdd(&sh.count[(k - mn) >> shift], 1);
    });
    lds_barrier();
    int x[4], sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += x[e] = sh.count[4 * t + e];
    int before = block_scan(sum, total, sh.red);
    if (before < want && before + sum >= want) {
      int e = 0;
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (e == k && before + x[k] < want) {
          before += x[k];
          ++e;
        }
      sh.found[0] = 4 * t + e;
      sh.found[1] = before;
    }
    lds_barrier();
    lo = mn + ((u64)sh.found[0] << shift);
    hi = mx - lo > (1ull << shift) - 1 ? lo + ((1ull << shift) - 1) : mx;
    want -= sh.found[1];
    if (shift == 0) {
      cut = lo;
      ties = want;
      break;
    }
    if (sh.count[sh.found[0]] <= 64) {  // each with all of them
      each(r, [&](int, u64 k) {
        if (k >= lo && k <= hi) sh.few[atomicAdd(&sh.n_few, 1)] = k;
      });
      lds_barrier();
      const int m = sh.n_few;
      if (t < m) {
        const u64 k = sh.few[t];
        int nb = 0, nt = 0;
#pragma unroll 4
        for (int j = 0; j < m; ++j) {
          nb += sh.few[j] < k;
          nt += sh.few[j] == k;
        }
        if (nb < want && nb + nt >= want) {  // (equal ones write the same)
          sh.ext[0][0] = k;
          sh.found[0] = want - nb;
        }
      }
      lds_barrier();
      cut = sh.ext[0][0];
      ties = sh.found[0];
      break;
    }
  }
  // eight columns a thread
  constexpr int E = 8;
  int at = 0;
  for (int c = 0; c < r.n; c += 256 * E) {
    const int j = c + E * t;
    u64 k[E];
    int id[E], tied = 0, under = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      k[e] = j + e < r.n ? r.at(j + e) : kNoPage;
      id[e] = j + e < r.n ? tab[j + e] : 0;
      tied += k[e] == cut;
      under += k[e] < cut;
    }
    int nt = 0, m, before = 0;
    if (ties != INT32_MAX) before = block_scan(tied, nt, sh.red);
    auto left = [&](int x) { return ties > x ? ties - x : 0; };
    int x = at + block_scan(under + (tied < left(before) ? tied : left(before)), m, sh.red);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool tie = k[e] == cut;
      if (k[e] < cut || (tie && before < ties)) to[x++] = id[e] * n_kv + g;
      before += tie;
    }
    at += m;
    ties = ties == INT32_MAX ? ties : left(nt);
  }
  return at;
}

// A work-group: `part` pages of one row and kv head; the last one of a row to arrive
// chooses. Grid: (parts, rows by kv heads), for several launches of the attention. Bound by
// latencies where rows are few: the row's place, its q, the pages' numbers, their bounds and what
// is handed over wait for each other (a row of 8 kv heads, 2047 pages: 16 us). Of many by the vector
// units, half of it the scores' conversions and products in 64 bits (300 rows of 4, 250 pages: 32).
template <int HD>
__global__ void __launch_bounds__(256) k_paged_select(SelectArgs s, int64_t row0, int part) {
  constexpr int LP = HD / 8, PAGES = 256 / LP;  // lanes that share a page, pages of a round
  __shared__ u64 key[kHeld];
  __shared__ int ids[kPart];
  __shared__ Choice sh;
  __shared__ int last;
  const PagedArgs &a = s.a;
  const int t = threadIdx.x, lane = t & 63;
  int at_row = blockIdx.y / a.n_kv, g = blockIdx.y % a.n_kv;
  if (a.row_start) {  // kv head by kv head within a launch of the attention
    const int first = at_row / s.rows * s.rows, left = gridDim.y / a.n_kv - first, rows = left < s.rows ? left : s.rows;
    const int x = blockIdx.y - first * a.n_kv;
    g = x / rows;
    at_row = first + x % rows;
  }
  const int64_t row = row0 + at_row;
  // its heads' q, on its way first
  const int l = lane % LP;
  const float *q = s.q + (row * s.n_head + (int64_t)g * s.group) * HD + 8 * l;
  constexpr int HU = 4;
  f32x4a4 y[HU][2];
  auto load_q = [&](int h0) {
#pragma unroll
    for (int h = 0; h < HU; ++h) {
      const float *p = q + (int64_t)(h0 + h < s.group ? h0 + h : 0) * HD;
      y[h][0] = *(const f32x4a4 *)p;
      y[h][1] = *(const f32x4a4 *)(p + 4);
    }
  };
  load_q(0);
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
  const int64_t cap = (int64_t)a.table_cols * a.page, pos = in ? (int64_t)a.seq_len[b] - n + row - r0 : -1;
  const int64_t end = pos + 1 < cap ? pos + 1 : cap;
  int32_t *to = s.table + (int64_t)blockIdx.y * s.n_select;
  if (end <= 0) {
    if (blockIdx.x == 0 && t == 0) {  // rows that no sequence has lie before the first and behind the last
      int64_t lo = 0, hi = 0, m;
      if (!in) {
        paged_rows(a, 0, lo, m);
        paged_rows(a, a.n_seq - 1, hi, m);
        hi += m;
      }
      s.len[blockIdx.y] = in || (row >= lo && row < hi) ? 0 : -1;
    }
    return;
  }
  const int mine = (int)((end - 1) / a.page);  // the row's own column
  const int parts = mine / part + 1;
  if ((int)blockIdx.x >= parts) return;
  const int c0 = blockIdx.x * part, nc = c0 + part < mine ? part : mine - c0;  // to score: columns before its own
  const int32_t *tab = a.table + (int64_t)b * a.table_cols;
  auto page = [&](int c) {
    const int32_t id = tab[c];
    return id >= 0 && id < a.n_pages ? id : -1;
  };
  const int own_id = page(mine), own = own_id >= 0, first = s.n_first < mine ? s.n_first : mine;
  for (int c = t; c < part; c += 256) ids[c] = c < nc ? page(c0 + c) : -1;
  // the heads' positive and negative parts, summed
  double qp[8], qn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) qp[e] = qn[e] = 0.0;
  for (int h0 = 0; h0 < s.group; h0 += HU) {
    if (h0) load_q(h0);
#pragma unroll
    for (int h = 0; h < HU; ++h) {
      if (h0 + h >= s.group) break;
      const float v[8] = {y[h][0][0], y[h][0][1], y[h][0][2], y[h][0][3], y[h][1][0], y[h][1][1], y[h][1][2], y[h][1][3]};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double x = v[e];
        qp[e] += x > 0.0 ? x : x != x ? x : 0.0;
        qn[e] += x < 0.0 ? x : 0.0;
      }
    }
  }
  lds_barrier();
  constexpr int U = 4;
  for (int c = t / LP; c < nc; c += U * PAGES) {
    h8 lo[U], hi[U];
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      id[u] = c + u * PAGES < nc ? ids[c + u * PAGES] : -1;
      const uint16_t *bd = s.bounds + ((int64_t)(id[u] < 0 ? 0 : id[u]) * a.n_kv + g) * 2 * HD + 8 * l;
      lo[u] = *(const h8 *)bd;
      hi[u] = *(const h8 *)(bd + HD);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      double x = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) x = fma((double)(float)lo[u][e], qn[e], fma((double)(float)hi[u][e], qp[e], x));
      const u64 k = c0 + c + u * PAGES < first ? 0 : rank_of(group_sum_d<LP>(x));
      if (l == 0 && c + u * PAGES < nc) key[c + u * PAGES] = id[u] < 0 ? kNoPage : k;
    }
  }
  lds_barrier();
  bool held = true;
  u64 *all = s.scores + (int64_t)blockIdx.y * a.table_cols;
  if (parts > 1) {
    for (int c = t; c < nc; c += 256) __hip_atomic_store(all + c0 + c, key[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0) last = __hip_atomic_fetch_add(s.counters + blockIdx.y, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)parts - 1;
    __syncthreads();
    if (!last) return;
    if (t == 0) __hip_atomic_store(s.counters + blockIdx.y, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    held = mine <= kHeld;
    if (held) {
      each(Handed{all, mine}, [&](int c, u64 k) { key[c] = k; });
      lds_barrier();
    }
  }
  const int want = s.n_select - own;
  const int at = held ? choose(Held{key, mine}, want, tab, a.n_kv, g, to, sh) : choose(Handed{all, mine}, want, tab, a.n_kv, g, to, sh);
  if (t == 0) {
    if (own) to[at] = own_id * a.n_kv + g;
    s.len[blockIdx.y] = (int32_t)(at * (int64_t)a.page + (own ? end - (int64_t)mine * a.page : 0));
  }
}

// Rows by kv heads of a launch of the attention (its plan of more takes LDS that work-groups
// then lack) and of the choice's, or one row's where it has more kv heads.
constexpr int64_t kRowsAtOnce = 1024, kMostHeads = 4096;
constexpr int64_t kScores = (int64_t)1 << 22;  // ranks, and chosen pages, of a launch

}  // namespace

bool select_fits(int64_t table_cols, int n_kv) { return table_cols <= (int64_t)1 << 20 && table_cols * n_kv <= kScores; }
int select_counters() { return (int)kMostHeads; }
size_t select_ws_bytes() { return kScores * 8 + kScores * 4 + kMostHeads * 4; }

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
  // rows of a launch of the attention: as many launches as are needed, the rows in equal parts;
  // a launch of the choice is for as many of those as its workspace holds (300 rows of 4 kv
  // heads, 250 pages: 32 us, two of 22 for an attention's launch each)
  const int64_t fit = std::min(kMostHeads, kScores / a.table_cols) / a.n_kv;
  const int64_t most = std::max<int64_t>(1, std::min(kRowsAtOnce / a.n_kv, fit));
  const int64_t launches = (a.s_rows + most - 1) / most, rows = (a.s_rows + launches - 1) / launches;
  const int64_t at_once = std::max<int64_t>(1, fit / rows) * rows;
  SelectArgs s{a, bounds, q, n_head, group, n_sel, n_first, (int)rows, (uint64_t *)ws, (int32_t *)(ws + kScores * 8), nullptr, select_counters};
  s.len = s.table + kScores;
  for (int64_t i = 0; i < a.s_rows; i += rows) {
    const int n_rows = (int)std::min(rows, a.s_rows - i), n = n_rows * a.n_kv;
    const int64_t before = i % at_once * a.n_kv;
    if (before == 0) {
      const int64_t heads = std::min(at_once, a.s_rows - i) * a.n_kv;
      // few rows: more work-groups a row (1 row of 8 kv heads, 2047 pages: 24 us with 512 pages each, 17 with 128)
      const int each = heads * ((a.table_cols + kPart - 1) / kPart) < 512 ? kPart / 4 : kPart;
      const dim3 grid((unsigned)((a.table_cols + each - 1) / each), (unsigned)heads);
      if (a.hd == 64) KMOE_LAUNCH(k_paged_select<64>, grid, dim3(256), 0, st, s, i, each);
      else KMOE_LAUNCH(k_paged_select<128>, grid, dim3(256), 0, st, s, i, each);
    }
    PagedArgs p = a;
    p.n_kv = 1;
    p.n_pages = a.n_pages * a.n_kv;
    p.n_seq = n;
    p.table_cols = n_sel;
    p.s_rows = n;
    p.row_start = nullptr;
    p.seq_len = s.len + before;
    p.table = s.table + before * n_sel;
    const int64_t at = i * n_head * a.hd;
    // rows of a chunk choose many of the same pages: kv head by kv head, kept in the caches
    const hipError_t e = a.row_start ? launch_paged_attention_again(st, p, n_rows, q + at, group, out + at, part, counters)
                                     : launch_paged_attention(st, p, q + at, group, 0, 0, out + at, part, counters);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace kmoe
