// kmoe_paged_attn.hip — attention over the paged key-value cache.
#include <algorithm>
#include <type_traits>

#include "kmoe_device.h"
#include "kmoe_launch.h"
#include "kmoe_paged.h"

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
// NaN or an infinity reaches this row only if the row sees it.
template <int T, int HD>
__device__ void plain_head(const PagedArgs &a, int b, int g, const float *qp, const Visible &vis, float *out) {
  constexpr int PARTS = 256 / HD;
  __shared__ float qs[HD], w[256], red[4], sum[4], accs[PARTS][HD];
  const int t = here(threadIdx.x), wave = t >> 6, lane = t & 63;
  const int64_t bb = paged_block_bytes(T, a.page, HD);
  const float scale = 1.0f / sqrtf((float)HD);
  __syncthreads();
  if (t < HD) qs[t] = qp[t];
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  bool any = false;
  for (int64_t p0 = 0; p0 <= vis.pos; p0 += 256) {
    if (p0 >= vis.sink && p0 + 256 <= vis.lo) {  // between the first positions and the window
      p0 = vis.lo / 256 * 256 - 256;
      continue;
    }
    const int64_t p = p0 + t;
    const uint8_t *blk = vis(p) ? paged_block(a, bb, b, p, g) : nullptr;
    __syncthreads();  // qs, and the last block's w read
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
    const float e = blk ? expf(sc - mn) : -1.0f;  // -1: not seen
    w[t] = e;
    const float ws = group_sum<64>(blk ? e : 0.0f);
    if (lane == 0) sum[wave] = ws;
    any = __syncthreads_or(blk != nullptr) || any;
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
  }
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

// Four floats by agent-scope loads.
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f32x4 ld4_agent(const float *p) {
  const f32x2 a = __builtin_bit_cast(f32x2, __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  const f32x2 b = __builtin_bit_cast(f32x2, __hip_atomic_load((const uint64_t *)p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  return f32x4{a.x, a.y, b.x, b.y};
}
constexpr float kLo = 0x1p-12f;
constexpr int kTile = 32;  // positions per step of a wave
// The running maximum is moved only by scores that pass it by more than this (in
// units of log2 e): the weights are then at most 2^kLag, and O is seldom scaled.
constexpr float kLag = 4.0f;
constexpr float kUp = 0x1p10f;  // weights times kUp stay below 2^14 in f16
// Work-groups of a CU that the registers let reside.
constexpr int paged_occ(int hd, int c) { return hd == 64 ? (c == 1 ? 4 : 3) : (c == 1 ? 3 : 2); }

// A pair of f32 as two dwords of f16 pairs: hi, the nearest f16, and lo, the
// nearest f16 of 2^12 times what hi leaves: x = hi + lo * 2^-12 to 2^-23 of x for
// |x| in 2^-14..2^15 and to 2^-37 below that.
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
  // (f32 values from here on: a product before the call may otherwise be rounded
  // to f16 in one step for hi and in two for lo, and the two then disagree)
  asm("" : "+v"(a), "+v"(b));
  hi = __builtin_bit_cast(uint32_t, (h2){(_Float16)a, (_Float16)b});
  asm("" : "+v"(hi));  // one packed conversion; lo reads its halves
  const h2 h = __builtin_bit_cast(h2, hi);
  lo = __builtin_bit_cast(uint32_t, (h2){(_Float16)fmaf((float)h.x, -1.0f / kLo, a * (1.0f / kLo)),
                                         (_Float16)fmaf((float)h.y, -1.0f / kLo, b * (1.0f / kLo))});
}

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

// 16 bytes per lane; NT: the line is used whole by this load and by nobody else.
template <bool NT>
__device__ __forceinline__ u32x4 load16(const uint8_t *p) {
  if constexpr (NT) return __builtin_nontemporal_load((const u32x4 *)p);
  return *(const u32x4 *)p;
}

// A wave's share of 32 positions of K and of V, as loaded.
template <int T, int HD, bool NT>
struct Frags;
template <int HD, bool NT>
struct Frags<kPgF16, HD, NT> {
  u32x4 k[2][HD / 32], v[HD / 16];
  __device__ __forceinline__ void load_k(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *p = blk + (pp >> 5) * (64 * HD) + lane * 16;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < HD / 32; ++t) k[s][t] = load16<NT>(p + (s * (HD / 32) + t) * 1024);
  }
  __device__ __forceinline__ void load_v(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *p = blk + pg * HD * 2 + (pp >> 5) * (64 * HD) + lane * 16;
#pragma unroll
    for (int u = 0; u < HD / 16; ++u) v[u] = load16<NT>(p + u * 1024);
  }
  // V elements of the lane's positions that are in `m` only (bit j: position j of its eight)
  __device__ __forceinline__ void keep_v(uint32_t m) {
    u32x4 b;
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = ((m >> (2 * i)) & 1 ? 0xffffu : 0u) | ((m >> (2 * i + 1)) & 1 ? 0xffff0000u : 0u);
#pragma unroll
    for (int u = 0; u < HD / 16; ++u) v[u] &= b;
  }
};
template <int HD, bool NT>
struct Frags<kPgQ8, HD, NT> {
  u32x4 k[2][HD / 64], ks[2][HD / 64], v[HD / 32], vs[HD / 32];
  __device__ __forceinline__ void load_k(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *p = blk + (pp >> 5) * (32 * HD) + lane * 16;
    const uint8_t *d = blk + pg * HD + (pp >> 5) * (2 * HD) + (lane >> 4) * (HD / 4);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < HD / 64; ++t) {
        k[s][t] = load16<NT>(p + (s * (HD / 64) + t) * 1024);
        ks[s][t] = *(const u32x4 *)(d + s * HD + t * 16);
      }
  }
  __device__ __forceinline__ void load_v(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *h = blk + pg * HD + pg * (HD / 32) * 2;
    const uint8_t *p = h + (pp >> 5) * (32 * HD) + lane * 16;
    const uint8_t *d = h + pg * HD + (pp >> 5) * (2 * HD) + (lane >> 4) * (HD / 2);
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) {
      v[u] = load16<NT>(p + u * 1024);
      vs[u] = *(const u32x4 *)(d + u * 16);
    }
  }
  // (the quants are finite whatever the bytes; the scales need not be)
  __device__ __forceinline__ void keep_v(uint32_t m) {
    u32x4 b;
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = ((m >> (2 * i)) & 1 ? 0xffffu : 0u) | ((m >> (2 * i + 1)) & 1 ? 0xffff0000u : 0u);
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) vs[u] &= b;
  }
};

__device__ __forceinline__ float half_of(const u32x4 &x, int i) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(x[i >> 1] >> (16 * (i & 1))));
}

// Positions a column tile's rows see, in tiles of 32: tile v of vt is v below
// n_first (the first positions), first + (v - n_first) above.
struct Span {
  int n_first, first, vt;
  __device__ __forceinline__ int tile(int v) const { return v < n_first ? v : first + (v - n_first); }
};
__device__ __forceinline__ Span span_of(int64_t pos_lo, int64_t pos_hi, int64_t cap, int window, int sink) {
  const int64_t hi = pos_hi + 1 < cap ? pos_hi + 1 : cap;
  if (hi <= 0) return Span{0, 0, 0};
  const int t_hi = (int)((hi + kTile - 1) / kTile);
  if (window == 0) return Span{0, 0, t_hi};
  const int64_t lo = pos_lo - window + 1 > 0 ? pos_lo - window + 1 : 0;
  int t_lo = (int)(lo / kTile);
  t_lo = t_lo < t_hi ? t_lo : t_hi;
  const int s_hi = (int)(((sink < hi ? sink : hi) + kTile - 1) / kTile);
  const int n = s_hi < t_lo ? s_hi : t_lo;
  return Span{n, t_lo, n + t_hi - t_lo};
}

// How a call's work is shared out. A column tile is 16 C columns: the sequence's
// rows by the heads of the group, row-major. A unit is one kv head of two column
// tiles of a sequence, the i-th from the front and the i-th from the back: with a
// causal mask the tiles that the two see together are about the same for every
// i. All units' tiles of 32 positions, a unit's rounded up to fours (one per
// wave) and with kUnitCost for what a unit costs besides, lie in one line, and
// every work-group takes an equal stretch of it: segments of column tiles, at most
// two of them split with its neighbours. Every work-group forms the plan from the
// lengths, so the shares follow what a captured call finds when it is replayed.
constexpr int kUnitCost = 8;
constexpr int kMinShare = 8;  // tiles

struct SeqPlan {
  int n_ct, per;  // column tiles; tiles of the line per unit
  __device__ __forceinline__ int pairs() const { return (n_ct + 1) >> 1; }
};
__device__ __forceinline__ int round4(int x) { return (x + 3) & ~3; }
template <int COLS>
__device__ __forceinline__ SeqPlan seq_plan(int64_t n, int64_t len, int group, int64_t cap, int window, int sink) {
  SeqPlan r{((int)n * group + COLS - 1) / COLS, 0};
  if (r.n_ct == 0) return r;
  const int all = span_of(0, len - 1, cap, 0, 0).vt;  // of the last row without a window
  // most of a column tile, and most of two that are paired: their last rows lie
  // (n_ct - 1) COLS / group + COLS / group positions after the first row together
  int one = all;
  const int64_t base = len - n > 0 ? len - n : 0;
  int64_t two = (2 * base + (uint32_t)((r.n_ct + 1) * COLS) / (uint32_t)group + 3 + kTile - 1) / kTile + 2;
  two = two < 2 * (int64_t)all ? two : 2 * (int64_t)all;
  if (window) {
    const int64_t w = (int64_t)(sink + kTile - 1) / kTile + (window + (n < COLS ? n : COLS) + kTile - 2) / kTile + 1;
    one = w < one ? (int)w : one;
    two = two < 2 * w ? two : 2 * w;
  }
  // (each rounded up to fours, and a column tile that sees nothing takes a place too)
  r.per = kUnitCost + (r.n_ct == 1 ? round4(one > 0 ? one : 1) : round4((int)two) + 8);
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

// start[b] (b <= n_seq): the line's tiles before sequence b; lens[b]: its length.
template <int COLS>
__device__ void make_plan(const PagedArgs &a, int group, int64_t cap, int window, int sink, int64_t *start,
                          int32_t *lens, int64_t *red) {
  const int per = (a.n_seq + 255) / 256, b0 = threadIdx.x * per;
  auto space = [&](int b) -> int64_t {
    int64_t r0, n;
    paged_rows(a, b, r0, n);
    const int32_t len = a.seq_len[b];
    lens[b] = len;
    const SeqPlan s = seq_plan<COLS>(n, len, group, cap, window, sink);
    return (int64_t)s.pairs() * a.n_kv * s.per;
  };
  int64_t sum = 0, total;
  for (int b = b0; b < b0 + per && b < a.n_seq; ++b) sum += space(b);
  int64_t at = scan(sum, total, red);
  if (per == 1) {
    if (b0 < a.n_seq) start[b0] = at;
  } else {
    for (int b = b0; b < b0 + per && b < a.n_seq; ++b) {
      start[b] = at;
      at += space(b);
    }
  }
  if (threadIdx.x == 0) start[a.n_seq] = total;
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

// Work-group: four waves, one segment of a column tile at a time; wave w takes
// its tiles w, w + 4, ... (32 positions each) with its own running softmax, and
// the waves are merged through LDS.
//
// Per tile and wave, v_mfma_f32_16x16x32_f16 throughout:
//   scores S^T[position, column] = K . q^T: A = K tiles as they lie in the page,
//     B = q, scaled by a power of two per column to [2^14, 2^15) and split into
//     two f16 pieces (LDS). Lane (kg, column) ends with positions 4 kg .. 4 kg + 3
//     of each 16.
//   O^T[dim, column] += V^T . P: A = V tiles as they lie in the page, B = the
//     weights of the lane's own eight positions, times kUp, as two f16 pieces,
//     straight from the score registers.
// K and V (Q8_0: the quants) are exact in f16 and all sums are f32. Q8_0: a score
// is summed 32 dims at a time, one K step, and scaled by the position's scale of
// those; V's scales go into the weights before they are split, over a power of
// two that no scale so far has passed, per 32 dims.
// The running maximum is in units of log2 e.
template <int T, int HD, int C>
__global__ void __launch_bounds__(256, paged_occ(HD, C))
    k_paged_attn(PagedArgs a, const float *__restrict__ q, int nh, int window, int sink, float *__restrict__ part,
                 float *__restrict__ part_ml, uint32_t *counters, float *__restrict__ out) {
  constexpr int NT = HD / 32, NU = HD / 16, COLS = 16 * C, OROW = HD + 4;
  extern __shared__ int64_t start[];  // [n_seq + 1], then lens [n_seq]
  int32_t *lens = (int32_t *)(start + a.n_seq + 1);
  __shared__ union {
    u32x4 q[C][NT][2][64];
    float o[4][COLS][OROW];
    float f[4 * COLS * OROW];
  } L;
  __shared__ float fs_lds[COLS], m_lds[4][COLS], l_lds[4][COLS];
  __shared__ f32x4 grp[256];
  __shared__ int64_t red[4];
  __shared__ uint32_t bad_cols, arrived;
  const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = nh / a.n_kv, magic = 65536 / group + 1;  // x / group = x * magic >> 16 for x < 64
  const int64_t bb = paged_block_bytes(T, a.page, HD);
  const int64_t cap = (int64_t)a.table_cols * a.page;
  const int pshift = __builtin_ctz(a.page);
  make_plan<COLS>(a, group, cap, window, sink, start, lens, red);

  // this work-group's stretch of the line; neighbours in it share an XCD's L2
  const int64_t total = uniform64(start[a.n_seq]);
  const int rank = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  int64_t share = div64(total + gridDim.x - 1, gridDim.x);
  share = share < kMinShare ? kMinShare : share < 16 ? (share + 3) & ~(int64_t)3 : share;
  const int64_t x0 = rank * share, x1 = x0 + share < total ? x0 + share : total;
  int b = 0;
  if (x0 < x1)  // the last sequence that starts at or before x0
    for (int hi = a.n_seq; hi - b > 1;) {
      const int mid = (b + hi) >> 1;
      if (start[mid] <= x0) b = mid;
      else hi = mid;
    }
  b = __builtin_amdgcn_readfirstlane(b);

  for (int64_t x = x0; x < x1;) {
    while (uniform64(start[b + 1]) <= x) ++b;
    const int64_t sb = uniform64(start[b]);
    int64_t r0v, rnv;
    paged_rows(a, b, r0v, rnv);
    const int64_t r0 = __builtin_amdgcn_readfirstlane((int)r0v);
    const int n = __builtin_amdgcn_readfirstlane((int)rnv), len = __builtin_amdgcn_readfirstlane(lens[b]);
    const int n_cols = n * group;
    const SeqPlan plan = seq_plan<COLS>(n, len, group, cap, window, sink);
    const int64_t unit = div64(x - sb, plan.per);
    const int off = (int)(x - sb - unit * plan.per);
    const int g = (int)div64(unit, plan.pairs()), pair = (int)(unit - (int64_t)g * plan.pairs());
    auto span = [&](int ct) {
      const int c = ct * COLS, e = c + COLS < n_cols ? c + COLS : n_cols;
      return span_of(len - n + (int)((uint32_t)c / (uint32_t)group), len - n + (int)((uint32_t)(e - 1) / (uint32_t)group), cap,
                     window, sink);
    };
    const int ct_a = plan.n_ct - 1 - pair;
    const Span sp_a = span(ct_a);
    const int len_a = round4(sp_a.vt > 0 ? sp_a.vt : 1);
    const bool second = off >= len_a;
    const int ct = second ? pair : ct_a;
    const Span sp = second ? span(ct) : sp_a;
    const int extent = second && ct == ct_a ? 0 : sp.vt > 0 ? sp.vt : 1;  // (a middle column tile has no partner)
    const int at = second ? off - len_a : off;
    if (at >= extent) {  // what is left of the first part's fours, or of the unit
      x += (second ? plan.per : len_a) - off;
      continue;
    }
    const int64_t X = x - at;  // where the column tile lies in the line
    const int v_end = (int)(x1 - X < extent ? x1 - X : extent);
    const int w_first = (int)div64(X, share), n_seg = (int)div64(X + extent - 1, share) - w_first + 1;
    x = X + v_end;

    // columns c0 .. c0 + nv - 1; column c is row i0 + (h0 + c) / group, head (h0 + c) % group
    const int c0 = ct * COLS, nv = n_cols - c0 < COLS ? n_cols - c0 : COLS;
    const int i0 = (int)((uint32_t)c0 / (uint32_t)group), h0 = c0 - i0 * group;
    auto row_of = [&](int c) { return i0 + (((h0 + c) * magic) >> 16); };
    auto head_of = [&](int c) { return h0 + c - (((h0 + c) * magic) >> 16) * group; };
    const int pos0 = len - n;
    const int64_t pos_lo = pos0 + i0, pos_hi = pos0 + row_of(nv - 1);
    const int hi_pos = (int)(pos_hi + 1 < cap ? pos_hi + 1 : cap);  // the columns' positions end here
    const int lo_pos = window && pos_lo - window + 1 > 0 ? (int)(pos_lo - window + 1) : 0;
    const int v_last = v_end < sp.vt ? v_end : sp.vt;

    // q of column tile `wave` (in the other waves, of one of them) on its way first, then K and V
    const int cq = 16 * (wave % C) + c16, cv = cq < nv ? cq : nv - 1;
    const float *qp = q + ((r0 + row_of(cv)) * nh + (int64_t)g * group + head_of(cv)) * HD + 8 * kg;
    f32x4a4 y[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      y[t][0] = *(const f32x4a4 *)(qp + 32 * t);
      y[t][1] = *(const f32x4a4 *)(qp + 32 * t + 4);
    }
    __builtin_amdgcn_sched_barrier(0);
    const_i32 row = (const_i32)(uintptr_t)(a.table + (int64_t)b * a.table_cols);
    auto page_of = [&](int v) -> int { return v < v_last ? row[sp.tile(v) >> (pshift - 5)] : -1; };
    // the block of a tile's page (page 0 stands in for one that does not exist)
    auto block = [&](int id) { return a.pages + ((int64_t)id * a.n_kv + g) * bb; };
    auto exists = [&](int id) { return id >= 0 && id < a.n_pages; };
    Frags<T, HD, C == 1> fr;
    int v = at + wave;
    int id = page_of(v), id_next = page_of(v + 4);  // pages of the wave's tile and of its next one
    if (v < v_last) {
      const int pp = (sp.tile(v) * kTile) & (a.page - 1);
      const uint8_t *p = block(exists(id) ? id : 0);
      fr.load_k(p, a.page, pp, lane);
      fr.load_v(p, a.page, pp, lane);
    }
    __builtin_amdgcn_sched_barrier(0);
    {
      float amax = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(y[t][e >> 2][e & 3]));
      amax = quad_max(amax);
      int sh = 15 - ((int)(__float_as_uint(amax) >> 23) - 126);
      sh = sh < 100 ? sh : 100;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        u32x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t u, w;
          split2(ldexpf(y[t][e >> 1][2 * (e & 1)], sh), ldexpf(y[t][e >> 1][2 * (e & 1) + 1], sh), u, w);
          hi[e] = u;
          lo[e] = w;
        }
        if (wave < C) {
          L.q[wave % C][t][0][lane] = hi;
          L.q[wave % C][t][1][lane] = lo;
        }
      }
      if (wave < C && kg == 0)
        fs_lds[cq] = ldexpf((float)(1.4426950408889634 / (HD == 64 ? 8.0 : 11.313708498984761)), -sh);
    }
    // columns: position, first position of the window
    int pos_c[C], lo_c[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int cc = 16 * j + c16;
      const int64_t p = pos0 + row_of(cc < nv ? cc : nv - 1);
      pos_c[j] = cc < nv ? (int)(p < cap ? p : cap - 1) : -1;
      lo_c[j] = window && p - window + 1 > 0 ? (int)(p - window + 1) : 0;
    }
    lds_barrier();
    float fs[C];
    f32x4 O[C][NU];
    float m[C], l[C], up[T == kPgQ8 ? NT : 1], back[T == kPgQ8 ? NT : 1];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      fs[j] = fs_lds[16 * j + c16];
      m[j] = -INFINITY;
      l[j] = 0.0f;
#pragma unroll
      for (int u = 0; u < NU; ++u) O[j][u] = f32x4{0};
    }
    if constexpr (T == kPgQ8) {
#pragma unroll
      for (int u = 0; u < NT; ++u) up[u] = kUp * 0x1p24f, back[u] = 0x1p-24f;
    }

    // one tile; `more`: its registers are refilled with the wave's next one on the
    // way (a branch around the loads would make every wait one for all of them)
    auto step = [&](auto more) {
      const int p0 = sp.tile(v) * kTile;
      const bool ok = exists(id);
      const int pp_next = more ? (sp.tile(v + 4) * kTile) & (a.page - 1) : 0;
      const uint8_t *p_next = more ? block(exists(id_next) ? id_next : 0) : nullptr;
      id = id_next;
      id_next = page_of(v + 8);
      const int lq = here(lane);  // (q's pieces are read at each tile)
      // scores, in q's scale
      f32x4 S[C][2];
      if constexpr (T == kPgF16) {
        f32x4 lo[C][2], hi[C][2];
#pragma unroll
        for (int j = 0; j < C; ++j) lo[j][0] = lo[j][1] = hi[j][0] = hi[j][1] = f32x4{0};
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < C; ++j) {
            const h8 ql = __builtin_bit_cast(h8, L.q[j][t][1][lq]), qh = __builtin_bit_cast(h8, L.q[j][t][0][lq]);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const h8 k = __builtin_bit_cast(h8, fr.k[s][t]);
              lo[j][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql, lo[j][s], 0, 0, 0);
              hi[j][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh, hi[j][s], 0, 0, 0);
            }
          }
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[j][s][i] = fmaf(lo[j][s][i], kLo, hi[j][s][i]);
      } else {
#pragma unroll
        for (int j = 0; j < C; ++j) S[j][0] = S[j][1] = f32x4{0};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const h8 k = i8_h8(here(fr.k[s][t >> 1][2 * (t & 1)]), here(fr.k[s][t >> 1][2 * (t & 1) + 1]));
#pragma unroll
            for (int j = 0; j < C; ++j) {
              const h8 ql = __builtin_bit_cast(h8, L.q[j][t][1][lq]), qh = __builtin_bit_cast(h8, L.q[j][t][0][lq]);
              const f32x4 lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql, f32x4{0}, 0, 0, 0);
              const f32x4 hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh, f32x4{0}, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                S[j][s][i] = fmaf(fmaf(lo[i], kLo, hi[i]), half_of(fr.ks[s][t >> 1], 4 * (t & 1) + i), S[j][s][i]);
            }
          }
          __builtin_amdgcn_sched_barrier(0);  // (few registers rather than many products at once)
        }
      }
#pragma unroll
      for (int j = 0; j < C; ++j) asm volatile("" : "+v"(S[j][0]), "+v"(S[j][1]));  // formed before the loads
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (more) fr.load_k(p_next, a.page, pp_next, lane);
      // what some row does not see
      if (!ok || p0 + kTile > pos_lo + 1 || (window && p0 < (int)(pos_hi - window + 1) && p0 + kTile > sink)) {
        uint32_t keep = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int p = p0 + 16 * s + 4 * kg + i;
            if (ok && p < hi_pos && (p >= lo_pos || p < sink)) keep |= 1u << (4 * s + i);
#pragma unroll
            for (int j = 0; j < C; ++j)
              if (!(ok && p <= pos_c[j] && (p >= lo_c[j] || p < sink))) S[j][s][i] = -INFINITY;
          }
        fr.keep_v(keep);
      }
      if constexpr (T == kPgQ8) {  // V's largest scales so far
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          h2 d = {(_Float16)0.0f, (_Float16)0.0f};
#pragma unroll
          for (int i = 0; i < 4; ++i) d = __builtin_elementwise_max(d, __builtin_bit_cast(h2, fr.vs[u][i]));
          const float dm = fmaxf((float)d.x, (float)d.y);
          if (__builtin_amdgcn_ballot_w64(dm > back[u])) {
            const int ex = (int)(__float_as_uint(quad_max(dm)) >> 23) - 126;  // largest in [2^(ex - 1), 2^ex)
            const float r = ldexpf(back[u], -ex);  // O is kept times kUp / back
            back[u] = ldexpf(1.0f, ex);
            up[u] = ldexpf(kUp, -ex);
#pragma unroll
            for (int j = 0; j < C; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) O[j][2 * u][i] *= r, O[j][2 * u + 1][i] *= r;
          }
        }
      }
      // running softmax, and the weights' pieces
      float e8[C][8];
#pragma unroll
      for (int j = 0; j < C; ++j) {
        float mx = fmaxf(fmaxf(S[j][0][0], S[j][0][1]), fmaxf(S[j][0][2], S[j][0][3]));
        mx = fmaxf(mx, fmaxf(fmaxf(S[j][1][0], S[j][1][1]), fmaxf(S[j][1][2], S[j][1][3]))) * fs[j];
        if (__builtin_amdgcn_ballot_w64(mx > m[j] + kLag)) {
          mx = fmaxf(m[j], quad_max(mx));
          const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[j] - mx);
          m[j] = mx;
          l[j] *= f;
#pragma unroll
          for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) O[j][u][i] *= f;
        }
        const float mb = m[j] == -INFINITY ? 0.0f : m[j];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e8[j][i] = __builtin_amdgcn_exp2f(fmaf(S[j][i >> 2][i & 3], fs[j], -mb));
          sum += e8[j][i];
        }
        l[j] += sum;
      }
      // weighted V
      if constexpr (T == kPgF16) {
        u32x4 ph[C], pl[C];
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t y, z;
            split2(e8[j][2 * i] * kUp, e8[j][2 * i + 1] * kUp, y, z);
            ph[j][i] = y;
            pl[j][i] = z;
          }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const h8 y = __builtin_bit_cast(h8, fr.v[u]);
#pragma unroll
          for (int j = 0; j < C; ++j) {
            const f32x4 t = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, __builtin_bit_cast(h8, pl[j]), f32x4{0}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) O[j][u][i] = fmaf(t[i], kLo, O[j][u][i]);
            O[j][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, __builtin_bit_cast(h8, ph[j]), O[j][u], 0, 0, 0);
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const h8 y0 = i8_h8(here(fr.v[u][0]), here(fr.v[u][1])), y1 = i8_h8(here(fr.v[u][2]), here(fr.v[u][3]));
          float sc[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) sc[i] = half_of(fr.vs[u], i) * up[u];
#pragma unroll
          for (int j = 0; j < C; ++j) {
            u32x4 wh, wl;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t y, z;
              split2(e8[j][2 * i] * sc[2 * i], e8[j][2 * i + 1] * sc[2 * i + 1], y, z);
              wh[i] = y;
              wl[i] = z;
            }
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              const h8 y = d ? y1 : y0;
              const f32x4 t = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, __builtin_bit_cast(h8, wl), f32x4{0}, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i) O[j][2 * u + d][i] = fmaf(t[i], kLo, O[j][2 * u + d][i]);
              O[j][2 * u + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, __builtin_bit_cast(h8, wh), O[j][2 * u + d], 0, 0, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (more) fr.load_v(p_next, a.page, pp_next, lane);
      v += 4;
    };
    if (v < v_last) {
      while (v + 4 < v_last) step(std::true_type());
      step(std::false_type());
    }


    // the four waves' sums, O times kUp
    lds_barrier();  // every wave is done with q
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const float ls = quad_sum(l[j]);
      if (kg == 0) {
        m_lds[wave][16 * j + c16] = m[j];
        l_lds[wave][16 * j + c16] = ls;
      }
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        f32x4 y = O[j][u];
        if constexpr (T == kPgQ8)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] *= back[u >> 1];
        *(f32x4 *)&L.o[wave][16 * j + c16][16 * u + 4 * kg] = y;
      }
    }
    const int tl = here(tid);
    if (tl == 0) bad_cols = 0;
    lds_barrier();
    const bool whole = n_seg == 1;
    const int64_t my_slot = 2 * (int64_t)rank + (X >= x0);
    auto finish = [&](int c, int d, const f32x4 &y, float M, float Lsum) {
      const float inv = M == -INFINITY ? 0.0f : 1.0f / (kUp * Lsum);  // nothing seen: zeros
      const int i = row_of(c);
      bool fin = true;
      f32x4a4 r;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        r[k] = y[k] * inv;
        fin = fin && fabsf(r[k]) < INFINITY;
      }
      *(f32x4a4 *)(out + ((r0 + i) * nh + (int64_t)g * group + head_of(c)) * HD + d) = r;
      if (!fin || (M == -INFINITY && pos0 + i >= 0)) atomicOr(&bad_cols, 1u << c);
    };
    for (int e = tl; e < nv * (HD / 4); e += 256) {
      const int c = e / (HD / 4), d = e % (HD / 4) * 4;
      const float M = fmaxf(fmaxf(m_lds[0][c], m_lds[1][c]), fmaxf(m_lds[2][c], m_lds[3][c]));
      const float Mb = M == -INFINITY ? 0.0f : M;
      f32x4 y = f32x4{0};
      float Ls = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(m_lds[w][c] - Mb);
        Ls = fmaf(l_lds[w][c], f, Ls);
        const f32x4 z = *(const f32x4 *)&L.o[w][c][d];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = fmaf(z[i], f, y[i]);
      }
      if (whole) {
        finish(c, d, y, M, Ls);
      } else {
        float *op = part + (my_slot * COLS + c) * HD + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) st_agent(op + i, y[i]);
        if (d == 0) {
          st_agent(part_ml + (my_slot * COLS + c) * 2, M);
          st_agent(part_ml + (my_slot * COLS + c) * 2 + 1, Ls);
        }
      }
    }
    if (!whole) {
      // Hand over; the last work-group to arrive joins the segments, in their order.
      // What is handed over is written and read by agent-scope accesses only, which
      // gfx950 makes past the XCDs' L2s, and each wave has waited for its stores
      // (they are where every XCD reads them) before the barrier and the counter's
      // add. So the add needs no release of its own: that would write back the
      // XCD's whole L2, and with a work-group per slot of the chip it took 45 us
      // per launch (one row at 131000 positions 118 -> 96 us, 48 rows under a
      // window of 1024 68 -> 32).
      vm_wait();
      __syncthreads();
      const int tj = here(tid), lj = tj & 63;
            if (tj == 0) arrived = __hip_atomic_fetch_add(counters + w_first, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (arrived != (uint32_t)(n_seg - 1)) continue;
      auto slot = [&](int i) { return (int64_t)2 * (w_first + i) + (i == 0); };
      // each column's maximum, its segments' factors (LDS) and its sum: wave w columns w, w + 4, ...
      const int ns = n_seg;
      for (int c = wave; c < nv; c += 4) {
        float M = -INFINITY, Ls = 0.0f;
        for (int i = lj; i < ns; i += 64) M = fmaxf(M, ld_agent(part_ml + (slot(i) * COLS + c) * 2));
        M = group_max<64>(M);
        const float Mb = M == -INFINITY ? 0.0f : M;
        for (int i = lj; i < ns; i += 64) {
          const float f = __builtin_amdgcn_exp2f(ld_agent(part_ml + (slot(i) * COLS + c) * 2) - Mb);
          Ls = fmaf(ld_agent(part_ml + (slot(i) * COLS + c) * 2 + 1), f, Ls);
          L.f[i * COLS + c] = f;
        }
        Ls = group_sum<64>(Ls);
        if (lj == 0) {
          m_lds[0][c] = M;
          l_lds[0][c] = Ls;
        }
      }
      __syncthreads();
      // four dims per thread, the segments shared out among the threads that are left
      const int need = nv * (HD / 4), gs = need <= 128 ? 256 / need : 1;
      for (int e0 = 0; e0 < need; e0 += 256) {
        const int e = gs > 1 ? tj % need : e0 + tj, w = gs > 1 ? tj / need : 0;
        const int c = e / (HD / 4), d = e % (HD / 4) * 4;
        f32x4 y = f32x4{0};
        if (e < need && w < gs) {
          int i = w;
          for (; i + 7 * gs < ns; i += 8 * gs) {
            f32x4 z[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) z[k] = ld4_agent(part + (slot(i + k * gs) * COLS + c) * HD + d);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float f = L.f[(i + k * gs) * COLS + c];
#pragma unroll
              for (int t = 0; t < 4; ++t) y[t] = fmaf(z[k][t], f, y[t]);
            }
          }
          for (; i < ns; i += gs) {
            const f32x4 z = ld4_agent(part + (slot(i) * COLS + c) * HD + d);
            const float f = L.f[i * COLS + c];
#pragma unroll
            for (int t = 0; t < 4; ++t) y[t] = fmaf(z[t], f, y[t]);
          }
        }
        if (gs > 1) {
          grp[tj] = y;
          __syncthreads();
          for (int k = 1; w == 0 && k < gs; ++k)
#pragma unroll
            for (int t = 0; t < 4; ++t) y[t] += grp[tj + k * need][t];
        }
        if (e < need && w == 0) finish(c, d, y, m_lds[0][c], l_lds[0][c]);
      }
      if (tj == 0) st_agent(counters + w_first, 0u);  // zero again for the next call
    }
    lds_barrier();
    // an infinity or NaN among what a tile's columns see together spreads in the
    // products (0 * inf): such columns are formed again from their own positions,
    // as are those without a score above -inf (no page at all, or every score -inf)
    uint32_t bad = bad_cols;
    while (bad) {
      const int c = __builtin_ctz(bad);
      bad &= bad - 1;
      const int64_t at_row = (r0 + row_of(c)) * nh + g * group + head_of(c);
      plain_head<T, HD>(a, b, g, q + at_row * HD, visible_of(pos0 + row_of(c), window, sink), out + at_row * HD);
    }
    lds_barrier();
  }
}

}  // namespace

// Work-groups of a launch: as many as are resident at once on 256 CUs. (Twice as
// many, for an evener end: one row at 131000 positions 96 -> 106 us, 64 rows at
// 2000 95 -> 102, a prompt of 1777 rows 73 -> 104: more units are split.)
constexpr int paged_grid(int hd, int c) { return 256 * paged_occ(hd, c); }

size_t paged_part_floats() {
  size_t m = 0;
  for (int hd : {64, 128})
    for (int c : {1, 2}) m = std::max(m, (size_t)2 * paged_grid(hd, c) * 16 * c * (hd + 2));
  return m;
}
int paged_counters() { return paged_grid(64, 1); }

hipError_t launch_paged_attention(hipStream_t st, const PagedArgs &a, const float *q, int n_head, int64_t window,
                                  int64_t n_sink, float *out, float *part, uint32_t *counters) {
  const int group = n_head / a.n_kv;
  const int w = window >= INT32_MAX ? 0 : (int)window, sink = (int)(n_sink < (1 << 30) ? n_sink : (1 << 30));
  // 16 columns per tile where sequences have about one row
  const bool one = a.s_rows * group <= (int64_t)24 * a.n_seq;
  const int cols = one ? 16 : 32, most_wg = paged_grid(a.hd, one ? 1 : 2);
  // no more work-groups than the longest sequences that the table allows would fill
  const int64_t units = (a.s_rows * group / cols + a.n_seq) * a.n_kv;
  const int64_t most = units * (((int64_t)a.table_cols * a.page / kTile + kUnitCost + 3) / kMinShare + 1);
  const unsigned grid = (unsigned)std::min<int64_t>(most_wg, (most + 7) / 8 * 8);
  const size_t lds = (size_t)(a.n_seq + 1) * 8 + (size_t)a.n_seq * 4;
  float *ml = part + (size_t)2 * most_wg * cols * a.hd;
#define KMOE_PAGED(T, H, C) \
  KMOE_LAUNCH((k_paged_attn<T, H, C>), dim3(grid), dim3(256), lds, st, a, q, n_head, w, sink, part, ml, counters, out)
#define KMOE_PAGED_C(T, H)        \
  do {                            \
    if (one) KMOE_PAGED(T, H, 1); \
    else KMOE_PAGED(T, H, 2);     \
  } while (0)
  if (a.type == kPgF16) {
    if (a.hd == 64) KMOE_PAGED_C(kPgF16, 64);
    else KMOE_PAGED_C(kPgF16, 128);
  } else {
    if (a.hd == 64) KMOE_PAGED_C(kPgQ8, 64);
    else KMOE_PAGED_C(kPgQ8, 128);
  }
#undef KMOE_PAGED_C
#undef KMOE_PAGED
  return hipGetLastError();
}

}  // namespace kmoe
