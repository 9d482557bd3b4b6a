// kmoe_paged_attn.hip — attention over the paged key-value cache.
#include <algorithm>

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

// One row's head by a work-group of 256, in plain f32: 256 positions at a time,
// a thread per score, then a thread per dim (and 256 / HD parts of the
// positions), running maximum and sum. Every position is read by itself, so a
// NaN or an infinity reaches this row only if the row sees it.
template <int T, int HD>
__device__ void plain_head(const PagedArgs &a, int b, int g, const float *qp, const Visible &vis, float *out) {
  constexpr int PARTS = 256 / HD;
  __shared__ float qs[HD], w[256], red[4], sum[4], accs[PARTS][HD];
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
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

constexpr float kLo = 0x1p-12f;
constexpr int kTile = 32;  // positions per step of a wave

// A pair of f32 as two dwords of f16 pairs: hi, the nearest f16, and lo, the
// nearest f16 of 2^12 times what hi leaves: x = hi + lo * 2^-12 to 2^-23 of x for
// |x| in 2^-14..2^15 and to 2^-37 below that.
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
  // (f32 values from here on: a product before the call may otherwise be rounded
  // to f16 in one step for hi and in two for lo, and the two then disagree)
  asm("" : "+v"(a), "+v"(b));
  const h2 h = {(_Float16)a, (_Float16)b};
  const h2 l = {(_Float16)fmaf((float)h.x, -1.0f / kLo, a * (1.0f / kLo)),
                (_Float16)fmaf((float)h.y, -1.0f / kLo, b * (1.0f / kLo))};
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, l);
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

// A wave's share of 32 positions of K and of V, as loaded.
template <int T, int HD>
struct Frags;
template <int HD>
struct Frags<kPgF16, HD> {
  u32x4 k[2][HD / 32], v[HD / 16];
  __device__ __forceinline__ void load_k(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *p = blk + (pp >> 5) * (64 * HD) + lane * 16;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < HD / 32; ++t) k[s][t] = *(const u32x4 *)(p + (s * (HD / 32) + t) * 1024);
  }
  __device__ __forceinline__ void load_v(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *p = blk + pg * HD * 2 + (pp >> 5) * (64 * HD) + lane * 16;
#pragma unroll
    for (int u = 0; u < HD / 16; ++u) v[u] = *(const u32x4 *)(p + u * 1024);
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
template <int HD>
struct Frags<kPgQ8, HD> {
  u32x4 k[2][HD / 64], ks[2][HD / 64], v[HD / 32], vs[HD / 32];
  __device__ __forceinline__ void load_k(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *p = blk + (pp >> 5) * (32 * HD) + lane * 16;
    const uint8_t *d = blk + pg * HD + (pp >> 5) * (2 * HD) + (lane >> 4) * (HD / 4);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < HD / 64; ++t) {
        k[s][t] = *(const u32x4 *)(p + (s * (HD / 64) + t) * 1024);
        ks[s][t] = *(const u32x4 *)(d + s * HD + t * 16);
      }
  }
  __device__ __forceinline__ void load_v(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *h = blk + pg * HD + pg * (HD / 32) * 2;
    const uint8_t *p = h + (pp >> 5) * (32 * HD) + lane * 16;
    const uint8_t *d = h + pg * HD + (pp >> 5) * (2 * HD) + (lane >> 4) * (HD / 2);
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) {
      v[u] = *(const u32x4 *)(p + u * 1024);
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

// How a call's work is shared out. A unit is one kv head of one column tile (16 C
// columns: the sequence's rows by the heads of the group, row-major); its
// positions are cut into chunks of `tpc` tiles, and an item is one chunk. Every
// work-group forms the same plan from the lengths, so the shares follow what a
// captured call finds when it is replayed.
struct Plan {
  int tpc, items;
};
// Most tiles that a column tile of the sequence can see.
__device__ __forceinline__ int seq_tiles(const PagedArgs &a, int64_t n, int64_t len, int rows_per, int window, int sink) {
  if (n == 0) return 0;
  const int all = span_of(0, len - 1, (int64_t)a.table_cols * a.page, 0, 0).vt;
  if (window == 0) return all;
  const int64_t w = (int64_t)(sink + kTile - 1) / kTile + ((int64_t)window + rows_per + kTile - 2) / kTile + 1;
  return w < all ? (int)w : all;
}

// Exclusive scan of two counts over the work-group's threads.
__device__ __forceinline__ void scan2(int64_t &x, int64_t &y, int64_t &tx, int64_t &ty, int64_t (*red)[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t ix = x, iy = y;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t ux = __shfl_up(ix, d), uy = __shfl_up(iy, d);
    if (lane >= d) {
      ix += ux;
      iy += uy;
    }
  }
  __syncthreads();
  if (lane == 63) {
    red[wave][0] = ix;
    red[wave][1] = iy;
  }
  __syncthreads();
  x = ix - x;
  y = iy - y;
  tx = ty = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) {
      x += red[w][0];
      y += red[w][1];
    }
    tx += red[w][0];
    ty += red[w][1];
  }
}

// start[b], slot[b] (b <= n_seq): items and partial slots before sequence b.
template <int C>
__device__ Plan make_plan(const PagedArgs &a, int group, int window, int sink, int target, int *start, int *slot,
                          int64_t (*red)[2]) {
  const int per = (a.n_seq + 255) / 256, b0 = threadIdx.x * per;
  const int rows_per = (16 * C + group - 1) / group + 1;
  int64_t tiles = 0, units = 0, tt, tu;
  for (int b = b0; b < b0 + per && b < a.n_seq; ++b) {
    int64_t r0, n;
    paged_rows(a, b, r0, n);
    const int64_t u = (n * group + 16 * C - 1) / (16 * C) * a.n_kv;
    units += u;
    tiles += u * seq_tiles(a, n, a.seq_len[b], rows_per, window, sink);
  }
  scan2(tiles, units, tt, tu, red);
  // chunks that give the launch's work-groups one item each where the units leave room for that
  const int64_t room = tu < target / 2 ? target - tu : target / 2;
  int64_t tpc = (tt + room - 1) / room;
  tpc = (tpc + 3) / 4 * 4;
  if (tpc < 4) tpc = 4;
  if (tpc > (int64_t)1 << 26) tpc = (int64_t)1 << 26;
  int64_t items = 0, slots = 0, ti, ts;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t i = items, s = slots;
    for (int b = b0; b < b0 + per && b < a.n_seq; ++b) {
      int64_t r0, n;
      paged_rows(a, b, r0, n);
      const int64_t u = (n * group + 16 * C - 1) / (16 * C) * a.n_kv;
      const int vt = seq_tiles(a, n, a.seq_len[b], rows_per, window, sink);
      const int64_t nch = vt > tpc ? (vt + tpc - 1) / tpc : 1;
      if (pass) {
        start[b] = (int)i;
        slot[b] = (int)s;
      }
      i += u * nch;
      s += nch > 1 ? u * nch : 0;
    }
    if (!pass) {
      items = i;
      slots = s;
      scan2(items, slots, ti, ts, red);
    }
  }
  if (threadIdx.x == 0) start[a.n_seq] = (int)ti;
  __syncthreads();
  // (more items than rows and positions allow: row_start is not ascending, nothing is done)
  return Plan{__builtin_amdgcn_readfirstlane((int)tpc), __builtin_amdgcn_readfirstlane(ti < (1 << 30) ? (int)ti : 0)};
}

// Work-group: four waves, one item at a time; wave w takes the chunk's tiles w,
// w + 4, ... (32 positions each) with its own running softmax, and the waves are
// merged through LDS.
//
// Per tile and wave, v_mfma_f32_16x16x32_f16 throughout:
//   scores S^T[position, column] = K . q^T: A = K tiles as they lie in the page,
//     B = q, scaled by a power of two per column to [2^14, 2^15) and split into
//     two f16 pieces, in registers. Lane (kg, column) ends with positions 4 kg ..
//     4 kg + 3 of each 16.
//   O^T[dim, column] += V^T . P: A = V tiles as they lie in the page, B = the
//     weights of the lane's own eight positions, times 2^14, as two f16 pieces,
//     straight from the score registers.
// K and V (Q8_0: the quants) are exact in f16 and all sums are f32. Q8_0: a score
// is summed 32 dims at a time, one K step, and scaled by the position's scale of
// those; V's scales go into the weights before they are split, over the tile's
// largest (a power of two), once per 32 dims.
// Scores and the running maximum are in units of log2 e.
#ifndef KMOE_OCC1
#define KMOE_OCC1 2
#endif
template <int T, int HD, int C>
__global__ void __launch_bounds__(256, KMOE_OCC1)
    k_paged_attn(PagedArgs a, const float *__restrict__ q, int nh, int window, int sink, int target,
                 float *__restrict__ part, float *__restrict__ part_ml, uint32_t *counters, float *__restrict__ out) {
  constexpr int NT = HD / 32, NU = HD / 16, COLS = 16 * C, OROW = HD + 4;
  extern __shared__ int plan_lds[];  // [2][n_seq + 1]
  __shared__ __attribute__((aligned(16))) float o_lds[4][COLS][OROW];
  __shared__ float m_lds[4][COLS], l_lds[4][COLS];
  __shared__ int64_t red[4][2];
  __shared__ uint32_t bad_cols, arrived;
  int *start = plan_lds, *slot = plan_lds + a.n_seq + 1;
  const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = nh / a.n_kv;
  const int64_t bb = paged_block_bytes(T, a.page, HD);
  const int64_t cap = (int64_t)a.table_cols * a.page;
  const int pshift = __builtin_ctz(a.page);
  const Plan plan = make_plan<C>(a, group, window, sink, target, start, slot, red);

  for (int item = blockIdx.x; item < plan.items; item += gridDim.x) {
    // the item's sequence: the last one that starts at or before it
    int b = 0;
    for (int hi = a.n_seq; hi - b > 1;) {
      const int mid = (b + hi) >> 1;
      if (start[mid] <= item) b = mid;
      else hi = mid;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    int64_t r0v, nv_;
    paged_rows(a, b, r0v, nv_);
    const int64_t r0 = __builtin_amdgcn_readfirstlane((int)r0v), n = __builtin_amdgcn_readfirstlane((int)nv_);
    const int64_t len = __builtin_amdgcn_readfirstlane(a.seq_len[b]);
    const int local = __builtin_amdgcn_readfirstlane(item - start[b]);
    const int n_ct = (int)((n * group + COLS - 1) / COLS);
    const int nch = __builtin_amdgcn_readfirstlane(start[b + 1] - start[b]) / (n_ct * a.n_kv);
    const int g = local % a.n_kv, ch = local / a.n_kv % nch;
    const int ct = n_ct - 1 - local / a.n_kv / nch;  // the later rows, which see more, first
    const int64_t c0 = (int64_t)ct * COLS;           // first column
    const int nv = (int)(n * group - c0 < COLS ? n * group - c0 : COLS);
    const int64_t i_lo = c0 / group, i_hi = (c0 + nv - 1) / group;
    const int64_t pos_lo = len - n + i_lo, pos_hi = len - n + i_hi;
    const Span sp = span_of(pos_lo, pos_hi, cap, window, sink);
    const int n_act = (sp.vt + plan.tpc - 1) / plan.tpc;
    if (ch >= n_act && !(ch == 0 && n_act == 0)) continue;
    const int v_end = (ch + 1) * plan.tpc < sp.vt ? (ch + 1) * plan.tpc : sp.vt;
    const int hi_pos = (int)(pos_hi + 1 < cap ? pos_hi + 1 : cap);  // positions of the item end here
    const int lo_pos = window && pos_lo - window + 1 > 0 ? (int)(pos_lo - window + 1) : 0;

    // columns: position, first position of the window, q in two pieces
    int pos_c[C], lo_c[C];
    float fs[C];
    h8 qh[C][NT], ql[C][NT];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int cc = 16 * j + c16, cv = cc < nv ? cc : nv - 1;
      const int64_t i = (c0 + cv) / group;
      const int h = (int)((c0 + cv) - i * group);
      const int64_t p = len - n + i;
      pos_c[j] = cc < nv ? (int)(p < cap ? p : cap - 1) : -1;
      lo_c[j] = window && p - window + 1 > 0 ? (int)(p - window + 1) : 0;
      const float *qp = q + ((r0 + i) * nh + (int64_t)g * group + h) * HD + 8 * kg;
      f32x4a4 x[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        x[t][0] = *(const f32x4a4 *)(qp + 32 * t);
        x[t][1] = *(const f32x4a4 *)(qp + 32 * t + 4);
      }
      float amax = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[t][e >> 2][e & 3]));
      amax = quad_max(amax);
      int sh = 15 - ((int)(__float_as_uint(amax) >> 23) - 126);
      sh = sh < 100 ? sh : 100;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        u32x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t y, z;
          split2(ldexpf(x[t][e >> 1][2 * (e & 1)], sh), ldexpf(x[t][e >> 1][2 * (e & 1) + 1], sh), y, z);
          hi[e] = y;
          lo[e] = z;
        }
        qh[j][t] = __builtin_bit_cast(h8, hi);
        ql[j][t] = __builtin_bit_cast(h8, lo);
      }
      fs[j] = ldexpf((float)(1.4426950408889634 / (HD == 64 ? 8.0 : 11.313708498984761)), -sh);
    }

    f32x4 O[C][NU];
    float m[C], l[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      m[j] = -INFINITY;
      l[j] = 0.0f;
#pragma unroll
      for (int u = 0; u < NU; ++u) O[j][u] = f32x4{0};
    }

    const_i32 row = (const_i32)(uintptr_t)(a.table + (int64_t)b * a.table_cols);
    // the block of a tile, and whether its page exists (page 0 stands in for one that does not)
    auto page_of = [&](int v) -> int { return v < v_end ? row[sp.tile(v) >> (pshift - 5)] : -1; };
    auto block = [&](int id) { return a.pages + ((int64_t)id * a.n_kv + g) * bb; };
    Frags<T, HD> fr;
    int v = ch * plan.tpc + wave;
    int id = page_of(v), id_next = page_of(v + 4);
    bool ok = id >= 0 && id < a.n_pages;
    if (v < v_end) {
      const int pp = (sp.tile(v) * kTile) & (a.page - 1);
      const uint8_t *p = block(ok ? id : 0);
      fr.load_k(p, a.page, pp, lane);
      fr.load_v(p, a.page, pp, lane);
    }
    for (; v < v_end; v += 4) {
      const int p0 = sp.tile(v) * kTile;
      const bool more = v + 4 < v_end;
      const bool ok_next = id_next >= 0 && id_next < a.n_pages;
      const int pp_next = more ? (sp.tile(v + 4) * kTile) & (a.page - 1) : 0;
      const uint8_t *p_next = block(ok_next ? id_next : 0);
      id_next = page_of(v + 8);
      // scores
      f32x4 S[C][2];
      if constexpr (T == kPgF16) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < C; ++j) {
            f32x4 lo = f32x4{0}, hi = f32x4{0};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const h8 x = __builtin_bit_cast(h8, fr.k[s][t]);
              lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ql[j][t], lo, 0, 0, 0);
              hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh[j][t], hi, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) S[j][s][i] = fmaf(lo[i], kLo, hi[i]) * fs[j];
          }
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < C; ++j) {
            f32x4 sum = f32x4{0};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const h8 x = i8_h8(fr.k[s][t >> 1][2 * (t & 1)], fr.k[s][t >> 1][2 * (t & 1) + 1]);
              f32x4 lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ql[j][t], f32x4{0}, 0, 0, 0);
              f32x4 hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh[j][t], f32x4{0}, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                sum[i] = fmaf(fmaf(lo[i], kLo, hi[i]), half_of(fr.ks[s][t >> 1], 4 * (t & 1) + i), sum[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) S[j][s][i] = sum[i] * fs[j];
          }
      }
      if (more) fr.load_k(p_next, a.page, pp_next, lane);
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
      // running softmax, and the weights' pieces
      u32x4 ph[C], pl[C];
      float e8[C][8];
#pragma unroll
      for (int j = 0; j < C; ++j) {
        float mx = fmaxf(fmaxf(S[j][0][0], S[j][0][1]), fmaxf(S[j][0][2], S[j][0][3]));
        mx = fmaxf(mx, fmaxf(fmaxf(S[j][1][0], S[j][1][1]), fmaxf(S[j][1][2], S[j][1][3])));
        mx = fmaxf(m[j], quad_max(mx));
        if (__builtin_amdgcn_ballot_w64(mx > m[j])) {
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
          e8[j][i] = __builtin_amdgcn_exp2f(S[j][i >> 2][i & 3] - mb);
          sum += e8[j][i];
        }
        l[j] += sum;
        if constexpr (T == kPgF16) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t x, y;
            split2(e8[j][2 * i] * 0x1p14f, e8[j][2 * i + 1] * 0x1p14f, x, y);
            ph[j][i] = x;
            pl[j][i] = y;
          }
        }
      }
      // weighted V
      if constexpr (T == kPgF16) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const h8 x = __builtin_bit_cast(h8, fr.v[u]);
#pragma unroll
          for (int j = 0; j < C; ++j) {
            f32x4 t = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(h8, pl[j]), f32x4{0}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] *= kLo;
            t = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(h8, ph[j]), t, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) O[j][u][i] += t[i];
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          // the tile's largest scale of these dims, as a power of two
          float dm = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) dm = fmaxf(dm, half_of(fr.vs[u], i));
          dm = quad_max(dm);
          int ex = (int)(__float_as_uint(dm) >> 23) - 126;  // dm in [2^(ex - 1), 2^ex)
          ex = dm > 0.0f ? ex : 0;
          const float up = ldexpf(1.0f, 14 - ex), back = ldexpf(1.0f, ex);
          const h8 x0 = i8_h8(fr.v[u][0], fr.v[u][1]), x1 = i8_h8(fr.v[u][2], fr.v[u][3]);
#pragma unroll
          for (int j = 0; j < C; ++j) {
            u32x4 wh, wl;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t x, y;
              split2(e8[j][2 * i] * (half_of(fr.vs[u], 2 * i) * up), e8[j][2 * i + 1] * (half_of(fr.vs[u], 2 * i + 1) * up), x, y);
              wh[i] = x;
              wl[i] = y;
            }
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              const h8 x = d ? x1 : x0;
              f32x4 t = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(h8, wl), f32x4{0}, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i) t[i] *= kLo;
              t = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(h8, wh), t, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i) O[j][2 * u + d][i] = fmaf(t[i], back, O[j][2 * u + d][i]);
            }
          }
        }
      }
      ok = ok_next;
      if (more) fr.load_v(p_next, a.page, pp_next, lane);
    }

    // the four waves' sums, O times 2^14
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const float ls = quad_sum(l[j]);
      if (kg == 0) {
        m_lds[wave][16 * j + c16] = m[j];
        l_lds[wave][16 * j + c16] = ls;
      }
#pragma unroll
      for (int u = 0; u < NU; ++u) *(f32x4 *)&o_lds[wave][16 * j + c16][16 * u + 4 * kg] = O[j][u];
    }
    if (tid == 0) bad_cols = 0;
    lds_barrier();
    const bool whole = n_act <= 1;
    const int unit_slot = slot[b] + ((n_ct - 1 - ct) * nch) * a.n_kv + g;  // of chunk 0; chunk i is i * n_kv further
    const int64_t my_slot = unit_slot + (int64_t)ch * a.n_kv;
    auto out_at = [&](int c) {
      const int64_t i = (c0 + c) / group;
      return out + ((r0 + i) * nh + (int64_t)g * group + (c0 + c - i * group)) * HD;
    };
    for (int e = tid; e < nv * (HD / 4); e += 256) {
      const int c = e / (HD / 4), d = e % (HD / 4) * 4;
      const float M = fmaxf(fmaxf(m_lds[0][c], m_lds[1][c]), fmaxf(m_lds[2][c], m_lds[3][c]));
      const float Mb = M == -INFINITY ? 0.0f : M;
      f32x4 x = f32x4{0};
      float L = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(m_lds[w][c] - Mb);
        L = fmaf(l_lds[w][c], f, L);
        const f32x4 y = *(const f32x4 *)&o_lds[w][c][d];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = fmaf(y[i], f, x[i]);
      }
      if (whole) {
        const float inv = M == -INFINITY ? 0.0f : 0x1p-14f / L;  // no position seen: zeros
        float *op = out_at(c) + d;
        bool fin = true;
        f32x4a4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = x[i] * inv;
          fin = fin && fabsf(y[i]) < INFINITY;
        }
        *(f32x4a4 *)op = y;
        if (!fin || (M == -INFINITY && len - n + (c0 + c) / group >= 0)) atomicOr(&bad_cols, 1u << c);
      } else {
        float *op = part + (my_slot * COLS + c) * HD + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) st_agent(op + i, x[i]);
        if (d == 0) {
          st_agent(part_ml + (my_slot * COLS + c) * 2, M);
          st_agent(part_ml + (my_slot * COLS + c) * 2 + 1, L);
        }
      }
    }
    if (!whole) {
      // hand over; the unit's last work-group to arrive joins its chunks, in their order
      vm_wait();
      __syncthreads();
      if (tid == 0) {
        arrived = add_release(counters + unit_slot, 1u);
        if (arrived == (uint32_t)(n_act - 1)) acquire_agent();
      }
      __syncthreads();
      if (arrived != (uint32_t)(n_act - 1)) continue;
      acquire_agent();
      for (int e = tid; e < nv * (HD / 4); e += 256) {
        const int c = e / (HD / 4), d = e % (HD / 4) * 4;
        float M = -INFINITY;
        for (int i = 0; i < n_act; ++i) M = fmaxf(M, ld_agent(part_ml + ((unit_slot + (int64_t)i * a.n_kv) * COLS + c) * 2));
        const float Mb = M == -INFINITY ? 0.0f : M;
        f32x4 x = f32x4{0};
        float L = 0.0f;
        for (int i = 0; i < n_act; ++i) {
          const int64_t at = (unit_slot + (int64_t)i * a.n_kv) * COLS + c;
          const float f = __builtin_amdgcn_exp2f(ld_agent(part_ml + at * 2) - Mb);
          L = fmaf(ld_agent(part_ml + at * 2 + 1), f, L);
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = fmaf(ld_agent(part + at * HD + d + k), f, x[k]);
        }
        const float inv = M == -INFINITY ? 0.0f : 0x1p-14f / L;
        float *op = out_at(c) + d;
        bool fin = true;
        f32x4a4 y;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          y[k] = x[k] * inv;
          fin = fin && fabsf(y[k]) < INFINITY;
        }
        *(f32x4a4 *)op = y;
        if (!fin || (M == -INFINITY && len - n + (c0 + c) / group >= 0)) atomicOr(&bad_cols, 1u << c);
      }
      if (tid == 0) st_agent(counters + unit_slot, 0u);  // zero again for the next call
    }
    __syncthreads();
    // an infinity or NaN among what a tile's columns see together spreads in the
    // products (0 * inf): such columns are formed again from their own positions,
    // as are those without a score above -inf (no page at all, or every score -inf)
    uint32_t bad = bad_cols;
    while (bad) {
      const int c = __builtin_ctz(bad);
      bad &= bad - 1;
      const int64_t i = (c0 + c) / group;
      const int h = g * group + (int)(c0 + c - i * group);
      plain_head<T, HD>(a, b, g, q + ((r0 + i) * nh + h) * HD, visible_of(len - n + i, window, sink),
                        out + ((r0 + i) * nh + h) * HD);
    }
    __syncthreads();
  }
}

}  // namespace

// Work-groups of a launch (resident at once on the whole chip) and the most items
// they are given: one each where the units leave room.
constexpr int kPagedTarget[2] = {512, 512};

size_t paged_part_floats() {
  size_t m = 0;
  for (int c = 0; c < 2; ++c) m = std::max(m, (size_t)2 * kPagedTarget[c] * 16 * (c + 1) * (128 + 2));
  return m;
}
int paged_counters() { return 2 * kPagedTarget[0]; }

hipError_t launch_paged_attention(hipStream_t st, const PagedArgs &a, const float *q, int n_head, int64_t window,
                                  int64_t n_sink, float *out, float *part, uint32_t *counters) {
  const int group = n_head / a.n_kv;
  const int w = window >= INT32_MAX ? 0 : (int)window, sink = (int)(n_sink < (1 << 30) ? n_sink : (1 << 30));
  // 16 columns per item where sequences have about one row
  const bool one = a.s_rows * group <= (int64_t)24 * a.n_seq;
  const int cols = one ? 16 : 32, target = kPagedTarget[one ? 0 : 1];
  const int64_t units = (a.s_rows * group / cols + a.n_seq) * a.n_kv;
  const int64_t chunks = ((int64_t)a.table_cols * a.page / kTile + 3) / 4;  // most of a unit
  const unsigned grid = (unsigned)std::min<int64_t>(target, units * std::max<int64_t>(1, std::min<int64_t>(chunks, target)));
  const size_t lds = (size_t)2 * (a.n_seq + 1) * 4;
  float *ml = part + (size_t)2 * target * cols * a.hd;
#define KMOE_PAGED(T, H, C) \
  KMOE_LAUNCH((k_paged_attn<T, H, C>), dim3(grid), dim3(256), lds, st, a, q, n_head, w, sink, target, part, ml, counters, out)
#define KMOE_PAGED_C(T, H)     \
  do {                         \
    if (one) KMOE_PAGED(T, H, 1); \
    else KMOE_PAGED(T, H, 2);  \
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
