// kmoe_paged_attn.hip — attention over the paged key-value cache: decode steps,
// prompt chunks and both in one launch.
//
// What bounds it, with times at the sizes of the comments below (F16 pages of 64
// positions, heads of 128 unless said): one row per sequence reads every K and V
// once for all heads of a group, 64 rows at 100 .. 8192 positions 88 us = 5.6 TB/s
// of pages, one row at 131000 positions (8 kv heads) 95 us; with Q8_0 pages (half
// the bytes) the vector units, which make f16 of the quants: 65 us for 286 MB.
// Prompts are bound by the vector and matrix units together, which overlap little
// with two waves a SIMD (4096 rows, 32 heads over 8: 375 us, 730 Tflop/s of f16
// products, at 2.05 GHz; a wave's next scores beside its own softmax, in whatever
// order, gained nothing), short calls by latencies: 37 positions 8.6 us, of
// which 4 are the launch, 2 the plan and 1 the first loads.
#include <algorithm>
#include <type_traits>

#include "kmoe_launch.h"
#include "kmoe_paged_attn.h"

namespace kmoe {

namespace {

// 16 bytes per lane, each line whole by one load. ONCE: by one work-group only, past
// the caches' order of use (decode steps, 64 rows at 2000 positions 100 -> 90 us).
// Column tiles of many rows read the same pages (with it two chunks of 512 rows and
// seven single rows, Q8_0, 272 -> 303 us; 4096 rows 359 -> 385).
template <bool ONCE>
__device__ __forceinline__ u32x4 load16(const uint8_t *p) {
  if constexpr (ONCE) return __builtin_nontemporal_load((const u32x4 *)p);
  return *(const u32x4 *)p;
}

// A wave's share of 32 positions of K and of V, as loaded.
template <int T, int HD, bool ONCE>
struct Frags;
template <int HD, bool ONCE>
struct Frags<kPgF16, HD, ONCE> {
  u32x4 k[2][HD / 32], v[HD / 16];
  __device__ __forceinline__ void load_k(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *p = blk + (pp >> 5) * (64 * HD) + lane * 16;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < HD / 32; ++t) k[s][t] = load16<ONCE>(p + (s * (HD / 32) + t) * 1024);
  }
  __device__ __forceinline__ void load_v(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *p = blk + pg * HD * 2 + (pp >> 5) * (64 * HD) + lane * 16;
#pragma unroll
    for (int u = 0; u < HD / 16; ++u) v[u] = load16<ONCE>(p + u * 1024);
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
template <int HD, bool ONCE>
struct Frags<kPgQ8, HD, ONCE> {
  u32x4 k[2][HD / 64], ks[2][HD / 64], v[HD / 32], vs[HD / 32];
  __device__ __forceinline__ void load_k(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *p = blk + (pp >> 5) * (32 * HD) + lane * 16;
    const uint8_t *d = blk + pg * HD + (pp >> 5) * (2 * HD) + (lane >> 4) * (HD / 4);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < HD / 64; ++t) {
        k[s][t] = load16<ONCE>(p + (s * (HD / 64) + t) * 1024);
        ks[s][t] = *(const u32x4 *)(d + s * HD + t * 16);
      }
  }
  __device__ __forceinline__ void load_v(const uint8_t *blk, int pg, int pp, int lane) {
    const uint8_t *h = blk + pg * HD + pg * (HD / 32) * 2;
    const uint8_t *p = h + (pp >> 5) * (32 * HD) + lane * 16;
    const uint8_t *d = h + pg * HD + (pp >> 5) * (2 * HD) + (lane >> 4) * (HD / 2);
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) {
      v[u] = load16<ONCE>(p + u * 1024);
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

// Work-groups of a CU that the registers let reside.
constexpr int paged_occ(int hd, int c) { return hd == 64 ? (c == 1 ? 4 : 3) : (c == 1 ? 3 : 2); }

// (A unit of decode steps counts 8 tiles besides its own, 12 where they are half as
// large: 200 rows of heads of 64, Q8_0, 8 tiles 55.6 us, 12 54.4, 16 55.5; 200 rows of
// heads of 128, F16, 81, 83, 86.)
template <int HD, int COLS>
using Work = Shares<COLS, 4, (HD == 64 && COLS == 16 ? 12 : 8), 8, 24>;

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
// K (Q8_0: its quants) and V are exact in f16 and all sums are f32. Q8_0: a score
// is summed 32 dims at a time, one K step, and scaled by the position's scale of
// those; a value, eight bits times eleven, is the sum of two f16 exactly.
// The running maximum is in units of log2 e.
template <int T, int HD, int C>
__global__ void __launch_bounds__(256, paged_occ(HD, C))
    k_paged_attn(PagedArgs a, const float *__restrict__ q, int nh, int window, int sink, float *__restrict__ part,
                 float *__restrict__ part_ml, uint32_t *counters, float *__restrict__ out) {
  constexpr int NT = HD / 32, NU = HD / 16, COLS = 16 * C, OROW = HD + 4;
  extern __shared__ int64_t start[];  // [n_seq + 1], then the lengths [n_seq]
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
  const int group = nh / a.n_kv, magic = 65536 / group + 1;  // x / group = x * magic >> 16 for x < 4096
  const int64_t bb = paged_block_bytes(T, a.page, HD);
  const int pshift = __builtin_ctz(a.page);
  Cursor<Work<HD, COLS>> cur(a, nh, window, sink, start, (int32_t *)(start + a.n_seq + 1), red);
  const int64_t cap = cur.cap;

  // wave 3 finds the next segment while this one's first loads are on their way (all
  // waves at once, each segment on its turn: 200 rows, Q8_0, 64 -> 58 us)
  __shared__ Seg segs[2];
  auto find = [&](int i) {
    if (wave != 3) return;
    Seg s;
    if (!cur.next(s)) s.b = -1;
    if (lane == 0) segs[i] = s;
  };
  find(0);
  lds_barrier();
  for (int turn = 0;; turn ^= 1) {
    const Seg s_ = uniform(segs[turn]);
    if (s_.b < 0) break;
    const int b = s_.b, g = s_.g, nv = s_.nv, pos0 = s_.pos0, v_last = s_.v_last, n_seg = s_.n_seg, w_first = s_.w_first;
    const int64_t r0 = s_.r0;
    const Span sp = s_.sp;
    auto row_of = [&](int c) { return s_.i0 + (((s_.h0 + c) * magic) >> 16); };
    auto head_of = [&](int c) { return s_.h0 + c - (((s_.h0 + c) * magic) >> 16) * group; };
    const int64_t pos_lo = pos0 + s_.i0, pos_hi = pos0 + row_of(nv - 1);
    const int hi_pos = (int)(pos_hi + 1 < cap ? pos_hi + 1 : cap);  // the columns' positions end here
    const int lo_pos = window && pos_lo - window + 1 > 0 ? (int)(pos_lo - window + 1) : 0;

    // q on its way first, then K and V (every wave forms pieces of q, the first C store theirs)
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
    int v = s_.at + wave;
    int id = page_of(v), id_next = page_of(v + 4);  // pages of the wave's tile and of its next one
    if (v < v_last) {
      const int pp = (sp.tile(v) * kTile) & (a.page - 1);
      const uint8_t *p = block(exists(id) ? id : 0);
      fr.load_k(p, a.page, pp, lane);
      fr.load_v(p, a.page, pp, lane);
    }
    __builtin_amdgcn_sched_barrier(0);
    find(turn ^ 1);
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
          split2(ldexpf(y[t][e >> 1][2 * (e & 1)], sh), ldexpf(y[t][e >> 1][2 * (e & 1) + 1], sh), 1.0f, kLoUp, u, w);
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
    // the lane's columns: position, first position of the window
    int pos_c[C], lo_c[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int cc = 16 * j + c16;
      const int64_t p = pos0 + row_of(cc < nv ? cc : nv - 1);
      pos_c[j] = cc < nv ? (int)(p < cap ? p : cap - 1) : -1;
      lo_c[j] = window && p - window + 1 > 0 ? (int)(p - window + 1) : 0;
    }
    lds_barrier();
    float fs[C], m[C], l[C];
    f32x4 O[C][NU];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      fs[j] = fs_lds[16 * j + c16];
      m[j] = -INFINITY;
      l[j] = 0.0f;
#pragma unroll
      for (int u = 0; u < NU; ++u) O[j][u] = f32x4{0};
    }

    // one tile; `more`: its registers are refilled with the wave's next one on the
    // way (a branch around the loads would make every wait one for all of them)
    bool paged = false;  // some tile of the wave has a page
    auto step = [&](auto more) {
      const int p0 = sp.tile(v) * kTile;
      const bool ok = exists(id);
      paged |= ok;
      const int pp_next = more ? (sp.tile(v + 4) * kTile) & (a.page - 1) : 0;
      const uint8_t *p_next = more ? block(exists(id_next) ? id_next : 0) : nullptr;
      const int lq = here(lane);  // (q's pieces are read at each tile)
      // (Q8_0: the wave at its products goes first, the others have the quants and
      // the softmax to do: 4096 rows 560 -> 546 us; with F16 pages the same)
      if constexpr (T == kPgQ8) __builtin_amdgcn_s_setprio(1);
      // scores, in q's scale
      f32x4 S[C][2];
      // (q's pieces of the next 32 dims are on their way while these are multiplied)
      h8 x[2][C][2];
      auto read_q = [&](int t) {
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) x[t & 1][j][h] = __builtin_bit_cast(h8, L.q[j][t][h][lq]);
      };
      read_q(0);
      if constexpr (T == kPgF16) {
        f32x4 lo[C][2], hi[C][2];
#pragma unroll
        for (int j = 0; j < C; ++j) lo[j][0] = lo[j][1] = hi[j][0] = hi[j][1] = f32x4{0};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (t + 1 < NT) read_q(t + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < C; ++j) {
              const h8 k = __builtin_bit_cast(h8, fr.k[s][t]);
              lo[j][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, x[t & 1][j][1], lo[j][s], 0, 0, 0);
              hi[j][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, x[t & 1][j][0], hi[j][s], 0, 0, 0);
            }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[j][s][i] = fmaf(lo[j][s][i], 1.0f / kLoUp, hi[j][s][i]);
      } else {
#pragma unroll
        for (int j = 0; j < C; ++j) S[j][0] = S[j][1] = f32x4{0};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (t + 1 < NT) read_q(t + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const h8 k = i8_h8(here(fr.k[s][t >> 1][2 * (t & 1)]), here(fr.k[s][t >> 1][2 * (t & 1) + 1]));
            const h8 kl = k * (_Float16)(1.0f / kLoUp);  // (exact: whole numbers up to 127)
#pragma unroll
            for (int j = 0; j < C; ++j) {
              f32x4 y = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, x[t & 1][j][1], f32x4{0}, 0, 0, 0);
              y = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, x[t & 1][j][0], y, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i) S[j][s][i] = fmaf(y[i], half_of(fr.ks[s][t >> 1], 4 * (t & 1) + i), S[j][s][i]);
            }
          }
          __builtin_amdgcn_sched_barrier(0);  // (few registers rather than many products at once)
        }
      }
#pragma unroll
      for (int j = 0; j < C; ++j) asm volatile("" : "+v"(S[j][0]), "+v"(S[j][1]));  // formed before the loads
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (T == kPgQ8) __builtin_amdgcn_s_setprio(0);
      if constexpr (more) fr.load_k(p_next, a.page, pp_next, lane);
      // (here, as scalar loads and LDS reads are waited for together: at the tile's
      // start the first products waited for the page table)
      id = id_next;
      id_next = page_of(v + 8);
      __builtin_amdgcn_sched_barrier(0);
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
        float e8[8], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e8[i] = __builtin_amdgcn_exp2f(fmaf(S[j][i >> 2][i & 3], fs[j], -mb));
          sum += e8[i];
        }
        l[j] += sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x, z;
          split2(e8[2 * i], e8[2 * i + 1], kUp, kLoUp, x, z);
          ph[j][i] = x;
          pl[j][i] = z;
        }
      }
      // weighted V
      if constexpr (T == kPgQ8) __builtin_amdgcn_s_setprio(1);
      if constexpr (T == kPgF16) {
        // (four dim tiles at a time: no product waits for the one before it)
#pragma unroll
        for (int u0 = 0; u0 < NU; u0 += 4) {
          f32x4 t[4][C];
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < C; ++j)
              t[u][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, fr.v[u0 + u]),
                                                               __builtin_bit_cast(h8, pl[j]), f32x4{0}, 0, 0, 0);
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < C; ++j)
              O[j][u0 + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  __builtin_bit_cast(h8, fr.v[u0 + u]), __builtin_bit_cast(h8, ph[j]), O[j][u0 + u], 0, 0, 0);
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < C; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) O[j][u0 + u][i] = fmaf(t[u][j][i], 1.0f / kLoUp, O[j][u0 + u][i]);
        }
      } else {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const h8 x = i8_h8(here(fr.v[u >> 1][2 * (u & 1)]), here(fr.v[u >> 1][2 * (u & 1) + 1]));
          const h8 d = __builtin_bit_cast(h8, fr.vs[u >> 1]);
          const h8 vh = x * d, vl = __builtin_elementwise_fma(x, d, -vh);  // exact: eight bits by eleven
#pragma unroll
          for (int j = 0; j < C; ++j)
            O[j][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, __builtin_bit_cast(h8, ph[j]), O[j][u], 0, 0, 0);
#pragma unroll
          for (int j = 0; j < C; ++j)
            O[j][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, __builtin_bit_cast(h8, ph[j]), O[j][u], 0, 0, 0);
          f32x4 t[C];
#pragma unroll
          for (int j = 0; j < C; ++j)
            t[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, __builtin_bit_cast(h8, pl[j]), f32x4{0}, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < C; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) O[j][u][i] = fmaf(t[j][i], 1.0f / kLoUp, O[j][u][i]);
          if (u & 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (T == kPgQ8) __builtin_amdgcn_s_setprio(0);
      if constexpr (more) fr.load_v(p_next, a.page, pp_next, lane);
      v += 4;
    };
    if (v < v_last) {
      while (v + 4 < v_last) step(std::true_type());
      step(std::false_type());
    }

    // the four waves' sums, O times kUp; without a score above -inf the sum of weights
    // says instead whether there was a page, here and in what is handed over
    lds_barrier();  // every wave is done with q
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const float ls = quad_sum(l[j]);
      if (kg == 0) {
        m_lds[wave][16 * j + c16] = m[j];
        l_lds[wave][16 * j + c16] = m[j] == -INFINITY && paged ? ls + 1.0f : ls;
      }
#pragma unroll
      for (int u = 0; u < NU; ++u) *(f32x4 *)&L.o[wave][16 * j + c16][16 * u + 4 * kg] = O[j][u];
    }
    const int tl = here(tid);
    if (tl == 0) bad_cols = 0;
    lds_barrier();
    const bool whole = n_seg == 1;
    const int64_t my_slot = 2 * (int64_t)cur.rank + s_.first;
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
      if (!fin || (M == -INFINITY && Lsum > 0.0f && pos0 + i >= 0)) atomicOr(&bad_cols, 1u << c);
    };
    for (int e = tl; e < nv * (HD / 4); e += 256) {
      const int c = e / (HD / 4), d = e % (HD / 4) * 4;
      const float M = fmaxf(fmaxf(m_lds[0][c], m_lds[1][c]), fmaxf(m_lds[2][c], m_lds[3][c]));
      const float Mb = M == -INFINITY ? 0.0f : M;
      f32x4 y = f32x4{0};
      float Ls = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_lds[w][c] - Mb);
        Ls = fmaf(l_lds[w][c], f, Ls);
        const f32x4 z = *(const f32x4 *)&L.o[w][c][d];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = fmaf(z[i], f, y[i]);
      }
      if (whole) {
        finish(c, d, y, M, Ls);
      } else {
        float *op = part + (my_slot * COLS + c) * HD + d;
        st2_agent(op, f32x2{y[0], y[1]});
        st2_agent(op + 2, f32x2{y[2], y[3]});
        if (d == 0) st2_agent(part_ml + (my_slot * COLS + c) * 2, f32x2{M, Ls});
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
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      const int tj = here(tid);
      if (tj == 0) arrived = __hip_atomic_fetch_add(counters + w_first, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (arrived != (uint32_t)(n_seg - 1)) continue;
      auto slot = [&](int i) { return (int64_t)2 * (w_first + i) + (i == 0); };
      // each column's maximum and sum: JP threads per column, which take its segments in turn
      constexpr int JP = 256 / COLS;
      const int ns = n_seg, jc = tj / JP, jp = tj % JP;
      float M = -INFINITY, Ls = 0.0f;
      for (int i = jp; i < ns; i += JP) {
        const f32x2 ml = ld2_agent(part_ml + (slot(i) * COLS + jc) * 2);
        const float Mn = fmaxf(M, ml.x);
        const bool none = Mn == -INFINITY;
        Ls = fmaf(ml.y, none ? 1.0f : __builtin_amdgcn_exp2f(ml.x - Mn), Ls * (none ? 1.0f : __builtin_amdgcn_exp2f(M - Mn)));
        M = Mn;
      }
      const float Mc = group_max<JP>(M), Mb = Mc == -INFINITY ? 0.0f : Mc;
      Ls = group_sum<JP>(Ls * (Mc == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - Mb)));
      if (jp == 0) {
        m_lds[0][jc] = Mc;
        l_lds[0][jc] = Ls;
      }
      // four dims of R elements per thread, the segments shared out among the threads
      // that are left; eight loads on their way at a time. The segments' factors lie
      // in LDS, kF segments at a time.
      constexpr int kF = 4 * OROW;
      const int need = nv * (HD / 4);
      auto join = [&](auto r_, int gs) {
        constexpr int R = decltype(r_)::value, U = 8 / R;
        const int e = gs > 1 ? tj % need : tj, w = gs > 1 ? tj / need : 0;
        const float *op[R];
        int cs[R];
        f32x4 y[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int er = e + 256 * r < need ? e + 256 * r : need - 1;
          cs[r] = er / (HD / 4);
          op[r] = part + (int64_t)er * 4;
          y[r] = f32x4{0};
        }
        for (int i0 = 0; i0 < ns; i0 += kF) {
          const int i1 = i0 + kF < ns ? i0 + kF : ns;
          __syncthreads();
          for (int i = i0 + jp; i < i1; i += JP)
            L.f[(i - i0) * COLS + jc] = __builtin_amdgcn_exp2f(ld_agent(part_ml + (slot(i) * COLS + jc) * 2) - Mb);
          __syncthreads();
          if (w >= gs) continue;
          auto add = [&](auto u_, int i) {
            constexpr int N = decltype(u_)::value;
            f32x4 z[N][R];
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
              for (int r = 0; r < R; ++r) z[k][r] = ld4_agent(op[r] + slot(i + k * gs) * (COLS * HD));
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
              for (int r = 0; r < R; ++r) {
                const float f = L.f[(i - i0 + k * gs) * COLS + cs[r]];
#pragma unroll
                for (int t = 0; t < 4; ++t) y[r][t] = fmaf(z[k][r][t], f, y[r][t]);
              }
          };
          int i = i0 + w;
          for (; i + (U - 1) * gs < i1; i += U * gs) add(std::integral_constant<int, U>(), i);
          for (; i < i1; i += gs) add(std::integral_constant<int, 1>(), i);
        }
        if (gs > 1) {
          grp[tj] = y[0];
          __syncthreads();
          for (int k = 1; w == 0 && k < gs; ++k)
#pragma unroll
            for (int t = 0; t < 4; ++t) y[0][t] += grp[tj + k * need][t];
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (e + 256 * r < need && w == 0) finish(cs[r], (e + 256 * r) % (HD / 4) * 4, y[r], m_lds[0][cs[r]], l_lds[0][cs[r]]);
      };
      if (need <= 128) join(std::integral_constant<int, 1>(), 256 / need);
      else join(std::integral_constant<int, COLS * HD / 1024>(), 1);
      if (tj == 0) st_agent(counters + w_first, 0u);  // zero again for the next call
    }
    lds_barrier();
    // an infinity or NaN among what a tile's columns see together spreads in the
    // products (0 * inf): such columns are formed again from their own positions,
    // as are those without a score above -inf where their sequence has a page (every
    // score -inf, or no page that the row sees)
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
// 2000 95 -> 102: more units are split.)
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
  // 16 columns per tile where sequences have few rows: at 32 columns each 36 us with
  // 16, 23 with 32 (16 sequences of 2000 positions, Q8_0, heads of 64); decode steps
  // of 8 heads would leave three quarters of 32 idle
  const bool one = a.s_rows * group <= (int64_t)24 * a.n_seq;
  const int cols = one ? 16 : 32, full = paged_grid(a.hd, one ? 1 : 2);
  // no more work-groups than the longest sequences that the table allows would fill
  const int64_t units = (a.s_rows * group / cols + a.n_seq) * a.n_kv;
  const int cost = one && a.hd == 64 ? Work<64, 16>::cost : Work<128, 16>::cost;
  const int64_t most = units * (((int64_t)a.table_cols * a.page / kTile + cost) / Work<64, 16>::least + 2);
  const unsigned grid = (unsigned)std::min<int64_t>(full, (most + 7) / 8 * 8);
  const size_t lds = (size_t)(a.n_seq + 1) * 8 + (size_t)a.n_seq * 4;
  float *ml = part + (size_t)2 * full * cols * a.hd;
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
