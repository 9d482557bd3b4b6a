// kmoe_paged.hip — rows into and out of the paged key-value cache, and page
// copies.
#include "kmoe_device.h"
#include "kmoe_launch.h"
#include "kmoe_paged.h"

namespace kmoe {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

// x / d to the nearest whole number within -127..127, ties to even, as if divided
// exactly: x times a reciprocal may land on the wrong side of a half; the remainder
// x - n d (d has 11 bits and n 8, so one fma forms it) says which. inv: 1 / d to an
// ulp or two.
__device__ __forceinline__ float round_quot(float x, float d, float inv) {
  const float y = x * inv;
  if (!(fabsf(y) < 127.0f)) return copysignf(127.0f, y);
  const float n = rintf(y), r = fmaf(-n, d, x), h = 0.5f * d;
  const bool odd = (int)n & 1;
  return n + (r > h || (r == h && odd) ? 1.0f : 0.0f) - (-r > h || (-r == h && odd) ? 1.0f : 0.0f);
}

// Q8_0 of four values among the eight lanes of a group of 32: the group's f16 scale
// is amax / 127, the quants are rounded against that scale. A scale past f16's range
// is its largest value (the quants saturate); a group that holds a NaN or an
// infinity gets a NaN scale and zero quants, so its positions read as NaN.
__device__ __forceinline__ uint32_t q8_of(const f32x4 &x, _Float16 &scale) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : INFINITY);
  amax = group_max<8>(amax);
  if (amax == INFINITY) {
    scale = __builtin_bit_cast(_Float16, (uint16_t)0x7e00);
    return 0;
  }
  const float d = amax / 127.0f;
  scale = d >= 65504.0f ? (_Float16)65504.0f : (_Float16)d;
  const float f = (float)scale;
  if (f == 0.0f) return 0;
  const float inv = __builtin_amdgcn_rcpf(f);
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= ((uint32_t)(int)round_quot(x[i], f, inv) & 0xffu) << (8 * i);
  return r;
}

// The 32 positions of one V tile and two K tiles, which a work-group handles: rows
// r of the tile sit at positions 32 tile + r and are rows i0 + r of sequence b,
// where those are rows of the call. Work-groups are counted along the rows: a
// sequence of n rows lies in at most n / 32 + 2 tiles.
struct RowTile {
  int b;
  int64_t r0, n, i0, tile;
  int lo, hi;  // its rows are lo .. hi - 1
  __device__ __forceinline__ bool has(int r) const { return r >= lo && r < hi; }
};
__device__ __forceinline__ bool row_tile(const PagedArgs &a, int64_t at, RowTile &t) {
  int64_t local = 0;
  t.b = (int)at;
  if (a.row_start) {
    auto key = [&](int b) { return (int64_t)(a.row_start[b] >> 5) + 2 * b; };
    int lo = 0, hi = a.n_seq;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (key(mid) <= at) lo = mid;
      else hi = mid;
    }
    t.b = lo;
    local = at - key(lo);
  }
  paged_rows(a, t.b, t.r0, t.n);
  const int64_t pos0 = (int64_t)a.seq_len[t.b] - t.n;
  t.tile = (pos0 >> 5) + local;
  t.i0 = 32 * t.tile - pos0;
  if (t.i0 <= -32 || t.i0 >= t.n) return false;
  t.lo = t.i0 < 0 ? (int)-t.i0 : 0;
  t.hi = t.n - t.i0 < 32 ? (int)(t.n - t.i0) : 32;
  return true;
}
unsigned row_tiles(const PagedArgs &a) {
  return (unsigned)(a.row_start ? (a.s_rows >> 5) + 2 * (int64_t)a.n_seq : (int64_t)a.n_seq);
}

constexpr int kQHeads = 8, kQRows = 8;  // of a work-group that rotates q

// Work-group (tile of 32 positions, kv head, K or V): the tile's rows turned through
// LDS into the page's pieces of 16 bytes (a K piece belongs to one position; a V
// piece to eight, and is stored whole where the call has all of them). Behind them,
// work-groups of kQHeads heads by kQRows rows rotate q. A thread's values are all on
// their way before the angles are formed; sincosf of a row's angles is what costs
// most. 1777 rows, 16 heads over 4, Q8_0: 12 us for 38 MB (a work-group of all 32
// rows and 2 heads of q: 17); a copy of as many bytes takes 7.
template <int T, int HD>
__global__ void __launch_bounds__(256) k_paged_store(PagedArgs a, const float *__restrict__ q, int64_t q_stride,
                                                     const float *__restrict__ k, int64_t k_stride,
                                                     const float *__restrict__ v, int64_t v_stride, int nh, int rd,
                                                     const float *__restrict__ inv_freq, int neox,
                                                     float *__restrict__ q_out) {
  constexpr int ROW = HD + 8;  // halves (or bytes) of a row in LDS
  constexpr int Q4 = HD / 4, N = HD / 32;  // fours of a row; fours of a thread and head: of rows tid / Q4 + 32 j / N
  __shared__ float2 rot[32][64];
  __shared__ __attribute__((aligned(16))) uint16_t tile[32][ROW];
  __shared__ _Float16 scales[32][4];
  RowTile rt;
  if (!row_tile(a, blockIdx.x, rt)) return;
  constexpr int hd = HD;
  const int half = rd / 2, tid = threadIdx.x, c = tid % Q4 * 4;
  auto row_at = [&](int j) { return tid / Q4 + j * (32 / N); };
  auto source = [&](int j) {  // (the first row of the call stands in for those that it has not)
    const int r = row_at(j);
    return rt.r0 + rt.i0 + (rt.has(r) ? r : rt.lo);
  };
  // the other four of a pair's dims: the same four where pairs are neighbours, and
  // where the halves' border lies inside a four (element by element then)
  const bool whole = neox && (half & 3) == 0;
  const int other = whole && c < rd ? (c < half ? c + half : c - half) : c;
  auto angles = [&](int row0, int rows) {
    for (int e = tid; e < rows * half; e += 256) {
      const int r = row0 + e / half, i = e % half;
      if (!rt.has(r)) continue;
      float sn, cs;
      sincosf((float)(32 * rt.tile + r) * inv_freq[i], &sn, &cs);
      rot[r][i] = make_float2(cs, sn);
    }
    __syncthreads();
  };
  auto rotate = [&](f32x4 x, const f32x4 &y, const float *row, int r) {
    if (c >= rd) return x;
    if (whole) {
      const bool low = c < half;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 z = rot[r][(low ? c : c - half) + e];
        x[e] = low ? x[e] * z.x - y[e] * z.y : y[e] * z.y + x[e] * z.x;
      }
    } else if (neox) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = c + e;
        if (i >= rd) continue;
        const bool low = i < half;
        const float2 z = rot[r][low ? i : i - half];
        const float o = row[low ? i + half : i - half];
        x[e] = low ? x[e] * z.x - o * z.y : o * z.y + x[e] * z.x;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        if (c + e >= rd) continue;
        const float2 z = rot[r][(c + e) >> 1];
        const float x0 = x[e], x1 = x[e + 1];
        x[e] = x0 * z.x - x1 * z.y;
        x[e + 1] = x0 * z.y + x1 * z.x;
      }
    }
    return x;
  };
  if ((int)blockIdx.y >= 2 * a.n_kv) {
    const int part = (int)blockIdx.y - 2 * a.n_kv, row0 = part % (32 / kQRows) * kQRows, h0 = part / (32 / kQRows) * kQHeads;
    if (row0 >= rt.hi || row0 + kQRows <= rt.lo) return;
    constexpr int M = kQRows * kQHeads * Q4 / 256;
    f32x4 x[M], y[M];
    auto at = [&](int j, int &r, int &h) {
      const int i = tid / Q4 + j * (256 / Q4);
      r = row0 + i / kQHeads;
      h = h0 + i % kQHeads;
    };
#pragma unroll
    for (int j = 0; j < M; ++j) {
      int r, h;
      at(j, r, h);
      const int64_t i = rt.i0 + (rt.has(r) ? r : row0 > rt.lo ? row0 : rt.lo);
      const float *row = q + (rt.r0 + i) * q_stride + (int64_t)(h < nh ? h : h0) * HD;
      x[j] = *(const f32x4a4 *)(row + c);
      y[j] = *(const f32x4a4 *)(row + other);
    }
    angles(row0, kQRows);
#pragma unroll
    for (int j = 0; j < M; ++j) {
      int r, h;
      at(j, r, h);
      if (h >= nh || !rt.has(r)) continue;
      const int64_t s = rt.r0 + rt.i0 + r;
      *(f32x4a4 *)(q_out + (s * nh + h) * HD + c) = rotate(x[j], y[j], q + s * q_stride + (int64_t)h * HD, r);
    }
    return;
  }
  const bool kv = (int)blockIdx.y >= a.n_kv;  // V
  const int g = kv ? (int)blockIdx.y - a.n_kv : (int)blockIdx.y;
  const float *in = (kv ? v : k) + (int64_t)g * HD;
  const int64_t stride = kv ? v_stride : k_stride;
  f32x4 x[N], y[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float *row = in + source(j) * stride;
    x[j] = *(const f32x4a4 *)(row + c);
    y[j] = *(const f32x4a4 *)(row + (kv ? c : other));
  }
  uint8_t *blk = paged_block(a, paged_block_bytes(T, a.page, HD), rt.b, 32 * rt.tile, g);
  if (!blk) return;
  const int p0 = (int)(32 * rt.tile) & (a.page - 1);
  if (!kv) angles(0, 32);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int r = row_at(j);
    const f32x4 z = kv ? x[j] : rotate(x[j], y[j], in + source(j) * stride, rt.has(r) ? r : rt.lo);
    if constexpr (T == kPgF16) {
      typedef _Float16 h4 __attribute__((ext_vector_type(4)));
      *(h4 *)&tile[r][c] = h4{(_Float16)z[0], (_Float16)z[1], (_Float16)z[2], (_Float16)z[3]};
    } else {
      _Float16 scale;
      *(uint32_t *)((uint8_t *)tile[r] + c) = q8_of(z, scale);
      if ((c & 31) == 0) scales[r][c >> 5] = scale;
    }
  }
  __syncthreads();
  if constexpr (T == kPgF16) {
    for (int e = tid; e < 4 * hd; e += 256) {
      uint8_t *to = blk + (kv ? paged_v_off<T>(a.page, hd, p0, 0) : paged_k_off<T>(hd, p0, 0)) + e * 16;
      if (!kv) {  // tile of 16 positions, 32 dims, 8 of them, position
        const int r = e / (2 * hd) * 16 + (e & 15), c = e % (2 * hd) / 64 * 32 + (e & 63) / 16 * 8;
        if (rt.has(r)) *(uint4 *)to = *(const uint4 *)&tile[r][c];
      } else {  // 16 dims, positions 4 j .. and 16 + 4 j .., dim
        const int c = e / 64 * 16 + (e & 15), r = (e & 63) / 16 * 4;
        uint16_t x[8];
        bool all = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int rj = r + (j & 3) + 4 * (j & 4);
          x[j] = tile[rj][c];
          all = all && rt.has(rj);
        }
        if (all) {
          *(uint4 *)to = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (rt.has(r + (j & 3) + 4 * (j & 4))) ((uint16_t *)to)[j] = x[j];
        }
      }
    }
  } else {
    for (int e = tid; e < 2 * hd; e += 256) {
      uint8_t *to = blk + (kv ? paged_v_off<T>(a.page, hd, p0, 0) : paged_k_off<T>(hd, p0, 0)) + e * 16;
      if (!kv) {  // tile of 16 positions, 64 dims, 8 of each 32, position
        const int r = e / hd * 16 + (e & 15), c = e % hd / 64 * 64 + (e & 63) / 16 * 8;
        if (rt.has(r)) {
          const uint2 x = *(const uint2 *)((const uint8_t *)tile[r] + c), y = *(const uint2 *)((const uint8_t *)tile[r] + c + 32);
          *(uint4 *)to = make_uint4(x.x, x.y, y.x, y.y);
        }
      } else {  // 32 dims, positions, dim and dim + 16
        const int c = e / 64 * 32 + (e & 15), r = (e & 63) / 16 * 4;
        uint8_t x[16];
        bool all = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int rj = r + (j & 3) + 4 * (j & 4);
          x[j] = ((const uint8_t *)tile[rj])[c];
          x[8 + j] = ((const uint8_t *)tile[rj])[c + 16];
          all = all && rt.has(rj);
        }
        if (all) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = x[4 * j] | x[4 * j + 1] << 8 | x[4 * j + 2] << 16 | (uint32_t)x[4 * j + 3] << 24;
          *(uint4 *)to = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (rt.has(r + (j & 3) + 4 * (j & 4))) to[j] = x[j], to[8 + j] = x[8 + j];
        }
      }
    }
    if (tid < hd) {  // 32 positions by hd / 32 groups
      const int r = tid & 31, u = tid >> 5;
      if (rt.has(r))
        *(_Float16 *)(blk + (kv ? paged_vs_off(a.page, hd, p0 + r, u) : paged_ks_off(a.page, hd, p0 + r, u))) = scales[r][u];
    }
  }
}

// The other way: work-group (tile, kv head) reads the pieces whole and writes rows.
template <int T, int HD>
__global__ void __launch_bounds__(256) k_paged_read(PagedArgs a, _Float16 *__restrict__ k, _Float16 *__restrict__ v) {
  constexpr int ROW = HD + 8;
  __shared__ __attribute__((aligned(16))) _Float16 tile[2][32][ROW];
  RowTile rt;
  if (!row_tile(a, blockIdx.x, rt)) return;
  constexpr int hd = HD;
  const int g = blockIdx.y, tid = threadIdx.x;
  const uint8_t *blk = paged_block(a, paged_block_bytes(T, a.page, hd), rt.b, 32 * rt.tile, g);
  const int p0 = (int)(32 * rt.tile) & (a.page - 1);
  if (blk) {
    const uint8_t *kp = blk + paged_k_off<T>(hd, p0, 0), *vp = blk + paged_v_off<T>(a.page, hd, p0, 0);
    if constexpr (T == kPgF16) {
      for (int e = tid; e < 4 * hd; e += 256) {
        const uint4 x = *(const uint4 *)(kp + e * 16), y = *(const uint4 *)(vp + e * 16);
        *(uint4 *)&tile[0][e / (2 * hd) * 16 + (e & 15)][e % (2 * hd) / 64 * 32 + (e & 63) / 16 * 8] = x;
        const int c = e / 64 * 16 + (e & 15), r = (e & 63) / 16 * 4;
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          tile[1][r + (j & 3) + 4 * (j & 4)][c] = __builtin_bit_cast(_Float16, (uint16_t)(w[j >> 1] >> (16 * (j & 1))));
      }
    } else {
      for (int e = tid; e < 2 * hd; e += 256) {
        const uint4 x = *(const uint4 *)(kp + e * 16), y = *(const uint4 *)(vp + e * 16);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
        const int r = e / hd * 16 + (e & 15), c = e % hd / 64 * 64 + (e & 63) / 16 * 8;
        const int vc = e / 64 * 32 + (e & 15), vr = (e & 63) / 16 * 4;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int cj = c + 32 * (j >> 3) + (j & 7), rj = vr + (j & 3) + 4 * (j & 4), wc = vc + 16 * (j >> 3);
          const float ks = (float)*(const _Float16 *)(blk + paged_ks_off(a.page, hd, p0 + r, cj >> 5));
          const float vs = (float)*(const _Float16 *)(blk + paged_vs_off(a.page, hd, p0 + rj, wc >> 5));
          tile[0][r][cj] = (_Float16)((float)(int8_t)(xs[j >> 2] >> (8 * (j & 3))) * ks);
          tile[1][rj][wc] = (_Float16)((float)(int8_t)(ys[j >> 2] >> (8 * (j & 3))) * vs);
        }
      }
    }
  }
  __syncthreads();
  const int q8 = hd / 8;
  for (int e = tid; e < 64 * q8; e += 256) {
    const int kv = e / (32 * q8), r = e / q8 & 31, c = e % q8 * 8;
    if (!rt.has(r)) continue;
    const uint4 x = blk ? *(const uint4 *)&tile[kv][r][c] : make_uint4(0, 0, 0, 0);
    typedef uint32_t u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));
    *(u32x4a2 *)((kv ? v : k) + ((rt.r0 + rt.i0 + r) * a.n_kv + g) * hd + c) = u32x4a2{x.x, x.y, x.z, x.w};
  }
}

// Pairs of pages per launch: they travel in the kernel's arguments, so a call
// needs no copy to the device and can be captured.
constexpr int kCopyPairs = 256;
struct CopyPairs {
  int32_t src[kCopyPairs], dst[kCopyPairs];
};
constexpr int kCopyPer = 4;  // 16-byte pieces per thread

// Grid (pieces of a page, pair, layer).
__global__ void __launch_bounds__(256) k_pages_copy(uint8_t *__restrict__ pages, int64_t layer_stride,
                                                    int64_t page_bytes, CopyPairs pairs) {
  uint8_t *base = pages + (int64_t)blockIdx.z * layer_stride;
  const uint8_t *s = base + pairs.src[blockIdx.y] * page_bytes;
  uint8_t *d = base + pairs.dst[blockIdx.y] * page_bytes;
  const int64_t o = ((int64_t)blockIdx.x * kCopyPer * 256 + threadIdx.x) * 16;
  uint4 x[kCopyPer];
#pragma unroll
  for (int i = 0; i < kCopyPer; ++i) {  // (past the end: the page's first piece, not stored)
    const int64_t at = o + i * 4096;
    x[i] = *(const uint4 *)(s + (at < page_bytes ? at : 0));
  }
#pragma unroll
  for (int i = 0; i < kCopyPer; ++i)
    if (o + i * 4096 < page_bytes) *(uint4 *)(d + o + i * 4096) = x[i];
}

}  // namespace

hipError_t launch_paged_store(hipStream_t st, const PagedArgs &a, const float *q, int64_t q_stride, const float *k,
                              int64_t k_stride, const float *v, int64_t v_stride, int n_head, int rope_dim,
                              const float *inv_freq, int neox, float *q_out) {
  const dim3 grid(row_tiles(a), (unsigned)(2 * a.n_kv + (n_head + kQHeads - 1) / kQHeads * (32 / kQRows)));
#define KMOE_STORE(T, H)                                                                                        \
  KMOE_LAUNCH((k_paged_store<T, H>), grid, dim3(256), 0, st, a, q, q_stride, k, k_stride, v, v_stride, n_head, \
              rope_dim, inv_freq, neox, q_out)
  if (a.type == kPgF16) {
    if (a.hd == 64) KMOE_STORE(kPgF16, 64);
    else KMOE_STORE(kPgF16, 128);
  } else {
    if (a.hd == 64) KMOE_STORE(kPgQ8, 64);
    else KMOE_STORE(kPgQ8, 128);
  }
#undef KMOE_STORE
  return hipGetLastError();
}

hipError_t launch_paged_read(hipStream_t st, const PagedArgs &a, uint16_t *k, uint16_t *v) {
  const dim3 grid(row_tiles(a), (unsigned)a.n_kv);
#define KMOE_READ(T, H) KMOE_LAUNCH((k_paged_read<T, H>), grid, dim3(256), 0, st, a, (_Float16 *)k, (_Float16 *)v)
  if (a.type == kPgF16) {
    if (a.hd == 64) KMOE_READ(kPgF16, 64);
    else KMOE_READ(kPgF16, 128);
  } else {
    if (a.hd == 64) KMOE_READ(kPgQ8, 64);
    else KMOE_READ(kPgQ8, 128);
  }
#undef KMOE_READ
  return hipGetLastError();
}

hipError_t launch_pages_copy(hipStream_t st, uint8_t *pages, int64_t n_layer, int64_t layer_stride,
                             int64_t page_bytes, const int32_t *src, const int32_t *dst, int64_t n) {
  constexpr int64_t per = (int64_t)kCopyPer * 256 * 16;
  for (int64_t at = 0; at < n; at += kCopyPairs) {
    CopyPairs p{};
    const int m = (int)(n - at < kCopyPairs ? n - at : kCopyPairs);
    for (int i = 0; i < m; ++i) {
      p.src[i] = src[at + i];
      p.dst[i] = dst[at + i];
    }
    const dim3 grid((unsigned)((page_bytes + per - 1) / per), (unsigned)m, (unsigned)n_layer);
    KMOE_LAUNCH(k_pages_copy, grid, dim3(256), 0, st, pages, layer_stride, page_bytes, p);
  }
  return hipGetLastError();
}

}  // namespace kmoe
