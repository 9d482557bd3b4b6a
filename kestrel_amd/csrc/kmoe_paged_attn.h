// kmoe_paged_attn.h — device code of the paged attention's kernel: the plain form
// of one row, splits for the f16 matrix cores, and how a call's work is shared out
// (internal).
#pragma once

#include "kmoe_device.h"
#include "kmoe_paged.h"
#include "kmoe_paged_walk.h"

namespace kmoe {
namespace {

// What row `pos` of a sequence sees: positions 0 .. pos, or with a window the
// last `window` of them and the first `sink`.
struct Visible {
  int64_t pos, lo, sink;  // lo <= p <= pos, or p < sink (and p <= pos)
  __device__ __forceinline__ bool operator()(int64_t p) const { return p <= pos && (p >= lo || p < sink); }
};
__device__ __forceinline__ Visible visible_of(int64_t pos, int64_t window, int64_t n_sink) {
  return Visible{pos, window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0, n_sink};
}

template <int T>
__device__ __forceinline__ float k_elem(const uint8_t *blk, int pg, int hd, int p, int d) {
  if constexpr (T == kPgF16) return (float)*(const _Float16 *)(blk + paged_k_off<T>(hd, p, d));
  return (float)*(const int8_t *)(blk + paged_k_off<T>(hd, p, d)) * (float)*(const _Float16 *)(blk + paged_ks_off(pg, hd, p, d >> 5));
}
template <int T>
__device__ __forceinline__ float v_elem(const uint8_t *blk, int pg, int hd, int p, int d) {
  if constexpr (T == kPgF16) return (float)*(const _Float16 *)(blk + paged_v_off<T>(pg, hd, p, d));
  return (float)*(const int8_t *)(blk + paged_v_off<T>(pg, hd, p, d)) * (float)*(const _Float16 *)(blk + paged_vs_off(pg, hd, p, d >> 5));
}

// x, as if first known here: what is formed of it is not formed earlier and held
// in registers.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// One row's head by a work-group of 256, in plain f32: 256 positions at a time,
// a thread per score, then a thread per dim (and 256 / HD parts of the
// positions), running maximum and sum. Every position is read by itself, so a
// NaN or an infinity reaches this row only if the row sees it. Stretches without pages
// are passed over.
template <int T, int HD>
__device__ void plain_head(const PagedArgs &a, int b, int g, const float *qp, const Visible &vis, float *out) {
  constexpr int PARTS = 256 / HD;
  __shared__ float qs[HD], w[256], red[4], sum[4], accs[PARTS][HD];
  __shared__ int held[4], nearest;
  const int t = here(threadIdx.x), wave = t >> 6, lane = t & 63;
  const int64_t bb = paged_block_bytes(T, a.page, HD);
  const float scale = 1.0f / sqrtf((float)HD);
  __syncthreads();
  if (t < HD) qs[t] = qp[t];
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  bool any = false;
  auto block = [&](int64_t p0) {
    const int64_t p = p0 + t;
    const uint8_t *blk = vis(p) ? paged_block(a, bb, b, p, g) : nullptr;
    const bool some = __builtin_amdgcn_ballot_w64(blk != nullptr);
    if (lane == 0) held[wave] = some;
    __syncthreads();  // (qs is there, too, and the last block's w read)
    if (!(held[0] | held[1] | held[2] | held[3])) return false;
    any = true;
    float sc = -INFINITY;
    if (blk) {
      const int pp = (int)(p % a.page);
      float s0 = 0.0f;
#pragma unroll 2
      for (int d = 0; d < HD; ++d) s0 = fmaf(qs[d], k_elem<T>(blk, a.page, HD, pp, d), s0);
      sc = s0 * scale;
    }
    const float wm = group_max<64>(sc);
    if (lane == 0) red[wave] = wm;
    __syncthreads();
    const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    const float f = m == mn ? 1.0f : expf(m - mn);
    const float mb = mn == -INFINITY ? 0.0f : mn;  // (scores of -inf alone, so far: they weigh nothing)
    const float e = blk ? expf(sc - mb) : -1.0f;  // -1: not seen
    w[t] = e;
    const float ws = group_sum<64>(blk ? e : 0.0f);
    if (lane == 0) sum[wave] = ws;
    __syncthreads();
    m = mn;
    l = l * f + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
    acc *= f;
    const int d = t % HD, j0 = t / HD * HD;
#pragma unroll 1
    for (int j = j0; j < j0 + HD; ++j) {
      const float e1 = w[j];
      if (e1 == -1.0f) continue;
      const uint8_t *vb = paged_block(a, bb, b, p0 + j, g);
      acc = fmaf(e1, v_elem<T>(vb, a.page, HD, (int)((p0 + j) % a.page), d), acc);
    }
    return true;
  };
  auto find = [&](int64_t col) {  // columns from col on that name no page, four a thread
    const int32_t *row = a.table + (int64_t)b * a.table_cols;
    __syncthreads();
    if (t == 0) nearest = 1024;
    __syncthreads();
    int n = 1024;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      const int64_t c = col + 256 * i + t, id = c < a.table_cols ? row[c] : -1;
      n = id >= 0 && id < a.n_pages ? 256 * i + t : n;
    }
    if (n < 1024) atomicMin(&nearest, n);
    __syncthreads();
    return nearest;
  };
  plain_walk(vis.pos, vis.lo, vis.sink, (int64_t)a.table_cols * a.page, a.page, block, find);
  __syncthreads();
  accs[t / HD][t % HD] = acc;
  __syncthreads();
  if (t < HD) {
    float o = 0.0f;
    for (int i = 0; i < PARTS; ++i) o += accs[i][t];
    out[t] = any ? o / l : 0.0f;
  }
}

// ---------------------------------------------------------------------------
// On the f16 matrix cores, with 32-bit arithmetic kept.

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef const int32_t __attribute__((address_space(4))) *const_i32;  // read through scalar loads

// Two or four floats by agent-scope accesses (8-byte aligned).
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void st2_agent(float *p, f32x2 v) {
  __hip_atomic_store((uint64_t *)p, __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 ld2_agent(const float *p) {
  return __builtin_bit_cast(f32x2, __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ f32x4 ld4_agent(const float *p) {
  const f32x2 a = ld2_agent(p), b = ld2_agent(p + 2);
  return f32x4{a.x, a.y, b.x, b.y};
}

constexpr int kTile = 32;  // positions per step of a wave
// The running maximum is moved only by scores that pass it by more than this (in
// units of log2 e): the weights are then at most 2^kLag, and O is seldom scaled.
constexpr float kLag = 4.0f;
constexpr float kUp = 0x1p11f;  // weights times kUp stay below 2^15 in f16

// A pair of f32 times a power of two as two dwords of f16 pairs: hi, the nearest
// f16, and lo, the nearest f16 of `lo_up` (a power of two) times what hi leaves:
// hi + lo / lo_up is off by 2^-23 of the product at most, and by 2^-25 / lo_up where
// that is less than it (the matrix cores take f16 subnormals as they are).
__device__ __forceinline__ void split2(float a, float b, float up, float lo_up, uint32_t &hi, uint32_t &lo) {
  // (f32 values from here on: a product before the call may otherwise be rounded
  // to f16 in one step for hi and in two for lo, and the two then disagree)
  asm("" : "+v"(a), "+v"(b));
  hi = __builtin_bit_cast(uint32_t, (h2){(_Float16)(a * up), (_Float16)(b * up)});
  asm("" : "+v"(hi));  // lo reads its halves
  const h2 h = __builtin_bit_cast(h2, hi);
  lo = __builtin_bit_cast(uint32_t, (h2){(_Float16)fmaf((float)h.x, -lo_up, a * (up * lo_up)),
                                         (_Float16)fmaf((float)h.y, -lo_up, b * (up * lo_up))});
}
// lo_up of q and of the weights: errors beside 2^-23 of 2^-48 of the largest weight (1;
// Q8_0: 2^-47, the product of what both first pieces leave) and 2^-52 of q's largest
// element. The products of the weights' lo have a sum of their own, joined tile by
// tile; q's lo has too on F16 pages, and on Q8_0 pages is multiplied by the quants /
// lo_up, exact in f16. (One sum for hi and an unscaled lo: 2^-36 and 2^-40, so that
// beside a first position with a zero value that takes all but e^-20 of the weight the
// others have seven bits. It took two chunks of 512 rows and seven single rows, Q8_0,
// 249 -> 234 us, 4096 rows, F16, 408 -> 385.)
constexpr float kLoUp = 0x1p12f;

// Largest of the four lanes l, l ^ 16, l ^ 32, l ^ 48 (a column's share of one
// score tile), and their sum.
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Four signed bytes as four f16: 1024 + (b + 128) has b + 128 in its low bits.
__device__ __forceinline__ void i8_f16(uint32_t x, uint32_t &a, uint32_t &b) {
  x ^= 0x80808080u;
  const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
  a = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - off);
  b = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - off);
}
__device__ __forceinline__ h8 i8_h8(uint32_t x, uint32_t y) {
  u32x4 r;
  uint32_t a, b;
  i8_f16(x, a, b);
  r[0] = a;
  r[1] = b;
  i8_f16(y, a, b);
  r[2] = a;
  r[3] = b;
  return __builtin_bit_cast(h8, r);
}

__device__ __forceinline__ float half_of(const u32x4 &x, int i) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(x[i >> 1] >> (16 * (i & 1))));
}

// Positions a column tile's rows see, in tiles of 32: tile v of vt is v below
// n_first (the first positions), first + (v - n_first) above.
struct Span {
  int n_first, first, vt;
  __device__ __forceinline__ int tile(int v) const { return v < n_first ? v : first + (v - n_first); }
};
__device__ __forceinline__ Span span_of(int64_t pos_lo, int64_t pos_hi, int64_t cap, int window, int sink, int skip = 0) {
  const int64_t hi = pos_hi + 1 < cap ? pos_hi + 1 : cap;
  if (hi <= 0) return Span{0, 0, 0};
  const int t_hi = (int)((hi + kTile - 1) / kTile);
  if (window == 0) return Span{0, skip, t_hi > skip ? t_hi - skip : 0};  // (skip: without a window only)
  const int64_t lo = pos_lo - window + 1 > 0 ? pos_lo - window + 1 : 0;
  int t_lo = (int)(lo / kTile);
  t_lo = t_lo < t_hi ? t_lo : t_hi;
  const int s_hi = (int)(((sink < hi ? sink : hi) + kTile - 1) / kTile);
  const int n = s_hi < t_lo ? s_hi : t_lo;
  return Span{n, t_lo, n + t_hi - t_lo};
}

// What a launch works: whole sequences; what the sequences of each group have in common
// (kShared: a group counts as a sequence, all its rows see all of it); or what is left of
// the sequences then (kOwn); or whole sequences that have pages in common (kAgain).
enum { kWhole = 0, kShared = 1, kOwn = 2, kAgain = 3 };
constexpr int kPlanners = 8;  // work-groups of kShared that work no tiles (one plans kOwn's): the others stay whole eights

// What a tile of 32 positions takes with 16 columns, and with 32, one against the other: the whole
// chip's time by the number of tiles, each kind as many at once as its registers allow (heads of
// 128, F16, 40000 of 16: 0.65 ns; 20000 of 32: 1.4).
constexpr int kWeight16 = 5, kWeight32 = 11;
__host__ __device__ __forceinline__ int tile_weight(int log_cols) { return log_cols == 4 ? kWeight16 : kWeight32; }

// Rows of group i together, its first sequence, its positions in common, and the weight that
// it saves per tile of those and kv head. Where that is not positive (rows that fill the
// column tiles anyway), or there is but one sequence, nothing is in common.
__device__ __forceinline__ int64_t group_rows(const PagedArgs &a, const SharedArgs &s, int i, int group, int &b0, int64_t &r0,
                                              int64_t &n, int64_t &len) {
  int lo = s.start[i], hi = s.start[i + 1];
  lo = lo < 0 ? 0 : lo;
  hi = hi < 0 ? 0 : hi < a.n_seq ? hi : a.n_seq;
  int32_t pages = s.pages[i];
  pages = pages < 0 ? 0 : pages < a.table_cols ? pages : a.table_cols;
  len = (int64_t)pages * a.page;
  b0 = lo;
  r0 = n = 0;
  if (hi - lo <= 1 || !pages) return 0;
  RowRange first, last;
  paged_rows(a, lo, first.r0, first.n);
  paged_rows(a, hi - 1, last.r0, last.n);
  const RowRange all = group_range(first, last);
  r0 = all.r0;
  n = all.n;
  if (!s.least) return 0;
  auto tiles = [&](int log) { return ((int)n * group + (1 << log) - 1) >> log; };
  const int seqs = hi - lo < (int)n ? hi - lo : (int)n, full = tiles(s.log_whole);  // (a sequence has a column tile at least)
  const int saved = (seqs > full ? seqs : full) * tile_weight(s.log_whole) - tiles(s.log_cols) * tile_weight(s.log_cols);
  if (saved <= 0) n = 0;
  return saved > 0 ? saved : 0;
}

// How a call's work is shared out. A column tile is COLS columns: the sequence's
// rows by the heads of the group, row-major. A unit is one kv head of two column
// tiles of a sequence, the i-th from the front and the i-th from the back: with a
// causal mask the tiles of 32 positions that the two see together are about the
// same for every i. All units' tiles, with `cost` for what a unit costs besides,
// lie in one line, and every work-group takes an equal stretch of it: segments of
// column tiles, at most two of them split with its neighbours. Every work-group
// forms the plan from the lengths, so the shares follow what a captured call finds
// when it is replayed.
template <int COLS_, int STEP_, int COST, int MIN, int WHOLE>
struct Shares {
  static constexpr int COLS = COLS_;
  static constexpr int STEP = STEP_;  // tiles that a work-group works at a time; a column tile takes a multiple
  static constexpr int cost = COST;
  static constexpr int least = MIN;   // tiles of a stretch
  static constexpr int whole = WHOLE; // tiles that a stretch may be longer by to hold whole units
  static __device__ __forceinline__ int up(int x) { return (x + STEP - 1) & ~(STEP - 1); }
};

struct SeqPlan {
  int n_ct, per, units;  // column tiles; tiles of the line per unit; units per kv head
};
template <class SH, int MODE>
__device__ __forceinline__ SeqPlan seq_plan(int64_t n, int64_t len, int group, int64_t cap, int window, int sink, int skip) {
  constexpr int COLS = SH::COLS;
  SeqPlan r{((int)n * group + COLS - 1) / COLS, 0, 0};
  if (r.n_ct == 0) return r;
  if constexpr (MODE == kShared) {  // every column tile sees everything: a unit of its own
    r.per = SH::cost + SH::up((int)(len / kTile));
    r.units = r.n_ct;
    return r;
  }
  r.units = (r.n_ct + 1) >> 1;
  const int all = span_of(0, len - 1, cap, 0, 0, skip).vt;  // of the last row without a window
  // most of a column tile, and most of two that are paired: their last rows lie
  // (n_ct - 1) COLS / group + COLS / group positions after the first row together
  int one = all;
  const int64_t base = len - n > 0 ? len - n : 0;
  int64_t two = (2 * base + (uint32_t)((r.n_ct + 1) * COLS) / (uint32_t)group + 3 + kTile - 1) / kTile + 2 - 2 * skip;
  two = two < 2 * (int64_t)all ? two : 2 * (int64_t)all;
  if (window) {
    const int64_t w = (int64_t)(sink + kTile - 1) / kTile + (window + (n < COLS ? n : COLS) + kTile - 2) / kTile + 1;
    one = w < one ? (int)w : one;
    two = two < 2 * w ? two : 2 * w;
  }
  // (each rounded up to whole steps, and a column tile that sees nothing takes a place too)
  r.per = SH::cost + (r.n_ct == 1 ? SH::up(one > 0 ? one : 1) : SH::up((int)two) + 2 * SH::STEP);
  return r;
}

// Exclusive scan over the work-group's threads, and the total.
__device__ __forceinline__ int64_t scan(int64_t x, int64_t &total, int64_t *red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t ix = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t ux = __shfl_up(ix, d);
    if (lane >= d) ix += ux;
  }
  if (lane == 63) red[wave] = ix;
  __syncthreads();
  x = ix - x;
  total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) x += red[w];
    total += red[w];
  }
  return x;
}

// The tiles that sequence b's group works of it, where all its rows lie behind that.
__device__ __forceinline__ int skip_of(const PagedArgs &a, const SharedArgs &sa, int group, int b) {
  int lo = 0;  // the last group that starts at or before b
  for (int hi = sa.n_group; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (sa.start[mid] <= b) lo = mid;
    else hi = mid;
  }
  int b0;
  int64_t r0, n, len, at, m;
  group_rows(a, sa, lo, group, b0, r0, n, len);
  paged_rows(a, b, at, m);
  const bool in = sa.start[lo] <= b && b < sa.start[lo + 1] && m > 0 && at >= r0 && at + m <= r0 + n;
  return in && (int64_t)a.seq_len[b] - m >= len ? (int)(len / kTile) : 0;
}

// start[b] (b <= n, the sequences or groups): the line's tiles before sequence b; lens[b]: its length, kOwn:
// lens[n + b]: the tiles of it that its group works (any: whether groups work anything).
// kShared: nothing at all where too little is saved.
template <class SH, int MODE>
__device__ void make_plan(const PagedArgs &a, const SharedArgs &sa, int n_seq, int group, int64_t cap, int window, int sink,
                          int64_t *start, int32_t *lens, int64_t *red, bool any = true) {
  const int per = (n_seq + 255) / 256, b0 = threadIdx.x * per;
  int64_t saved = 0;
  auto space = [&](int b) -> int64_t {
    int64_t r0, n, len;
    int skip = 0;
    if constexpr (MODE == kShared) {
      int first;
      saved += group_rows(a, sa, b, group, first, r0, n, len) * a.n_kv * (len / kTile);
    } else {
      paged_rows(a, b, r0, n);
      len = a.seq_len[b] > 0 ? a.seq_len[b] : 0;  // (a length below the rows leaves them nothing)
      if constexpr (MODE == kAgain) n = a.seq_len[b] >= 0;
      if constexpr (MODE == kOwn) {
        skip = any ? skip_of(a, sa, group, b) : 0;
        lens[n_seq + b] = skip;
      }
    }
    lens[b] = (int32_t)len;
    const SeqPlan s = seq_plan<SH, MODE>(n, len, group, cap, window, sink, skip);
    return (int64_t)s.units * a.n_kv * s.per;
  };
  if (n_seq == 1) {  // (no scan: 37 positions 9.3 -> 8.6 us)
    int64_t x = space(0);
    if (MODE == kShared && saved < sa.least) x = 0;
    if (threadIdx.x == 0) {
      start[0] = 0;
      start[1] = x;
    }
    __syncthreads();
    return;
  }
  int64_t sum = 0, total;
  for (int b = b0; b < b0 + per && b < n_seq; ++b) sum += space(b);
  int64_t at = scan(sum, total, red);
  if constexpr (MODE == kShared) {
    if (sa.least) {
      int64_t all;
      __syncthreads();  // (the first scan's sums are read)
      scan(saved, all, red);
      if (all < sa.least) total = 0;
    }
  }
  if (per == 1) {
    if (b0 < n_seq) start[b0] = at;
  } else {
    for (int b = b0; b < b0 + per && b < n_seq; ++b) {
      start[b] = at;
      at += space(b);
    }
  }
  if (threadIdx.x == 0) start[n_seq] = total;
  __syncthreads();
}

// x / d by 32 bits where x has no more.
__device__ __forceinline__ int64_t div64(int64_t x, int64_t d) {
  if (((uint64_t)x | (uint64_t)d) >> 32) return x / d;
  return (uint32_t)x / (uint32_t)d;
}
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32);
}

// A segment: tiles [at, v_last) of a column tile of sequence b, kv head g. Its
// columns are c0 .. c0 + nv - 1; column c is row i0 + (h0 + c) / group, head
// (h0 + c) % group of the sequence's rows.
struct Seg {
  int b, g, n, len, pos0;  // pos0: the position of row 0 (kShared: of every row); b: the sequence whose pages are read
  int r0;
  int nv, i0, h0;
  Span sp;
  int at, v_last;
  int w_first, n_seg;  // the stretches that the column tile lies in
  int first;           // it starts in this one
  int skip;            // tiles that the sequence's group works
};

// Of a segment that every lane reads at one place.
__device__ __forceinline__ Seg uniform(const Seg &x) {
  constexpr int W = sizeof(Seg) / 4;
  struct Words {
    int w[W];
  } r = __builtin_bit_cast(Words, x);
#pragma unroll
  for (int i = 0; i < W; ++i) r.w[i] = __builtin_amdgcn_readfirstlane(r.w[i]);
  return __builtin_bit_cast(Seg, r);
}

template <class SH, int MODE>
struct Cursor {
  const PagedArgs &a;
  const SharedArgs &sa;
  const int64_t *start;
  const int32_t *lens;
  int n_seq, group, window, sink, wgs, rank, b;
  int64_t cap, share, x0, x1, x;

  // This work-group's stretch; neighbours in the line share an XCD's L2.
  __device__ __forceinline__ Cursor(const PagedArgs &a_, const SharedArgs &sa_, int nh, int window_, int sink_,
                                    int64_t *start_, int32_t *lens_, int64_t *red)
      : a(a_), sa(sa_), start(start_), lens(lens_), n_seq(MODE == kShared ? sa_.n_group : a_.n_seq), group(nh / a_.n_kv),
        window(window_), sink(sink_), cap((int64_t)a_.table_cols * a_.page) {
    if constexpr (MODE == kOwn) {  // (a work-group of the launch before has made the plan: 64 rows behind 6000 positions 61 -> 57 us)
      for (int b = threadIdx.x; b < n_seq; b += 256) {
        const int64_t at = sa.plan[b];
        const int32_t len = sa.lens[b], skip = sa.lens[n_seq + b];
        start_[b] = at;
        lens_[b] = len;
        lens_[n_seq + b] = skip;
      }
      if (threadIdx.x == 0) start_[n_seq] = sa.plan[n_seq];
      __syncthreads();
    } else {
      make_plan<SH, MODE>(a, sa, n_seq, group, cap, window, sink, start_, lens_, red);
    }
    const int64_t total = uniform64(start[n_seq]);
    wgs = (int)gridDim.x - (MODE == kShared ? kPlanners : 0);
    rank = (int)(blockIdx.x & 7) * (wgs >> 3) + (int)(blockIdx.x >> 3);
    share = div64(total + wgs - 1, wgs);
    share = share < SH::least ? SH::least : share < 4 * SH::STEP ? SH::up((int)share) : share;
    // One sequence: whole units where they fill the work-groups about as well, a join
    // and the segments besides cost more than these tiles (1777 rows, 16 heads: 64 ->
    // 58 us; 4000 rows, 32 heads: 434 -> 380; twice that many tiles: 1200 rows, 32
    // heads, 66 -> 84). Where not all work-groups are needed, equal parts of a unit
    // (64 rows at 700 positions, 32 heads: 30 -> 23 us).
    if (MODE == kWhole && SH::COLS > 16 && n_seq == 1) {
      int64_t r0, n;
      paged_rows(a, 0, r0, n);
      const SeqPlan p = seq_plan<SH, MODE>(n, lens[0], group, cap, window, sink, 0);
      const int64_t units = (int64_t)p.units * a.n_kv;
      if (share <= SH::least) {
        const int parts = p.per / SH::least;
        if (parts) share = SH::up((p.per + parts - 1) / parts);
      } else {
        const int64_t each = div64(units + wgs - 1, wgs) * p.per;
        if (2 * units >= wgs && each <= share + SH::whole) share = each;
      }
    }
    x0 = rank * share;
    x1 = x0 + share < total ? x0 + share : total;
    x = x0;
    int lo = 0;
    if (x0 < x1)  // the last sequence that starts at or before x0
      for (int hi = n_seq; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x0) lo = mid;
        else hi = mid;
      }
    b = __builtin_amdgcn_readfirstlane(lo);
  }

  __device__ __forceinline__ bool next(Seg &s) {
    constexpr int COLS = SH::COLS;
    while (x < x1) {
      while (uniform64(start[b + 1]) <= x) ++b;
      const int64_t sb = uniform64(start[b]);
      s.b = b;
      s.skip = 0;
      if constexpr (MODE == kShared) {
        int64_t r0, n, len;
        group_rows(a, sa, b, group, s.b, r0, n, len);
        s.b = __builtin_amdgcn_readfirstlane(s.b);
        s.r0 = __builtin_amdgcn_readfirstlane((int)r0);
        s.n = __builtin_amdgcn_readfirstlane((int)n);
      } else if constexpr (MODE == kAgain) {
        s.r0 = b % sa.rows * (n_seq / sa.rows) + b / sa.rows;
        s.n = 1;  // (one without a row takes no place in the line)
      } else if (a.row_start) {
        const const_i32 rs = (const_i32)(uintptr_t)a.row_start + b;
        s.r0 = rs[0] < 0 ? 0 : rs[0];
        const int hi = rs[1] < (int)a.s_rows ? rs[1] : (int)a.s_rows;
        s.n = hi > (int)s.r0 ? hi - (int)s.r0 : 0;
      } else {
        s.r0 = b;
        s.n = b < a.s_rows ? 1 : 0;
      }
      s.len = __builtin_amdgcn_readfirstlane(lens[b]);
      if constexpr (MODE == kOwn) s.skip = __builtin_amdgcn_readfirstlane(lens[n_seq + b]);
      s.pos0 = MODE == kShared ? s.len - 1 : s.len - s.n;
      const int n_cols = s.n * group;
      const SeqPlan plan = seq_plan<SH, MODE>(s.n, s.len, group, cap, window, sink, s.skip);
      const int64_t unit = div64(x - sb, plan.per);
      const int off = (int)(x - sb - unit * plan.per);
      s.g = (int)div64(unit, plan.units);
      const int pair = (int)(unit - (int64_t)s.g * plan.units);
      auto span = [&](int ct) {
        if constexpr (MODE == kShared) return Span{0, 0, s.len / kTile};
        const int c = ct * COLS, e = c + COLS < n_cols ? c + COLS : n_cols;
        return span_of(s.pos0 + (int)((uint32_t)c / (uint32_t)group), s.pos0 + (int)((uint32_t)(e - 1) / (uint32_t)group),
                       cap, window, sink, s.skip);
      };
      const int ct_a = MODE == kShared ? pair : plan.n_ct - 1 - pair;
      const Span sp_a = span(ct_a);
      const int len_a = SH::up(sp_a.vt > 0 ? sp_a.vt : 1);
      const bool second = off >= len_a;
      const int ct = second ? pair : ct_a;
      s.sp = second ? span(ct) : sp_a;
      const int extent = second && ct == ct_a ? 0 : s.sp.vt > 0 ? s.sp.vt : 1;  // (a middle column tile has no partner)
      s.at = second ? off - len_a : off;
      if (s.at >= extent) {  // what is left of the first part's last step, or of the unit
        x += (second ? plan.per : len_a) - off;
        continue;
      }
      const int64_t X = x - s.at;  // where the column tile lies in the line
      const int v_end = (int)(x1 - X < extent ? x1 - X : extent);
      s.first = X >= x0;
      s.w_first = (int)div64(X, share);
      s.n_seg = (int)div64(X + extent - 1, share) - s.w_first + 1;
      s.v_last = v_end < s.sp.vt ? v_end : s.sp.vt;
      const int c0 = ct * COLS;
      s.nv = n_cols - c0 < COLS ? n_cols - c0 : COLS;
      s.i0 = (int)((uint32_t)c0 / (uint32_t)group);
      s.h0 = c0 - s.i0 * group;
      x = X + v_end;
      return true;
    }
    return false;
  }
};

}  // namespace
}  // namespace kmoe
