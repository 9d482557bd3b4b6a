// kmoe_paged.hip — rows into and out of the paged key-value cache, and page
// copies.
#include "kmoe_device.h"
#include "kmoe_launch.h"
#include "kmoe_paged.h"

namespace kmoe {

namespace {

// x / d to the nearest whole number within -127..127, ties to even, as if divided
// exactly: the quotient of f32 may land on the wrong side of a half by its own
// rounding; the remainder x - n d (d has 11 bits and n 8, so one fma forms it)
// says which.
__device__ __forceinline__ float round_quot(float x, float d) {
  const float y = x / d;
  if (!(fabsf(y) < 127.0f)) return copysignf(127.0f, y);
  float n = rintf(y);
  const float r = fmaf(-n, d, x), h = 0.5f * d;
  const bool odd = (int)n & 1;
  if (r > h || (r == h && odd)) n += 1.0f;
  else if (-r > h || (-r == h && odd)) n -= 1.0f;
  return n;
}

// Q8_0 of one value among 32 lanes: the block's f16 scale is amax / 127, the
// quants are rounded against that scale. A scale past f16's range is its largest
// value (the quants saturate); a block that holds a NaN or an infinity gets a
// NaN scale and zero quants, so its positions read as NaN.
__device__ __forceinline__ void q8_of(float x, int8_t &q, _Float16 &scale) {
  const bool bad = !(fabsf(x) < INFINITY);
  const float amax = group_max<32>(bad ? INFINITY : fabsf(x));
  if (amax == INFINITY) {
    scale = __builtin_bit_cast(_Float16, (uint16_t)0x7e00);
    q = 0;
    return;
  }
  const float d = amax / 127.0f;
  scale = d >= 65504.0f ? (_Float16)65504.0f : (_Float16)d;
  const float f = (float)scale;
  q = f > 0.0f ? (int8_t)round_quot(x, f) : (int8_t)0;
}

// Work-group (row, four heads): one wave per head of q (rotated into q_out), k
// (rotated, into its page) or v (into its page).
template <int T>
__global__ void __launch_bounds__(256) k_paged_store(PagedArgs a, const float *__restrict__ q, int64_t q_stride,
                                                     const float *__restrict__ k, int64_t k_stride,
                                                     const float *__restrict__ v, int64_t v_stride, int nh, int rd,
                                                     const float *__restrict__ inv_freq, int neox,
                                                     float *__restrict__ q_out) {
  __shared__ float sn[64], cs[64];
  const int64_t s = blockIdx.x;
  const int b = paged_seq_of(a, s);
  if (b < 0) return;
  int64_t r0, n;
  paged_rows(a, b, r0, n);
  const int64_t p = (int64_t)a.seq_len[b] - n + (s - r0);
  const int half = rd / 2, hd = a.hd;
  for (int i = threadIdx.x; i < half; i += 256) {
    float sv, cv;
    sincosf((float)p * inv_freq[i], &sv, &cv);
    sn[i] = sv;
    cs[i] = cv;
  }
  __syncthreads();
  const int head = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (head >= nh + 2 * a.n_kv) return;
  const bool is_q = head < nh, is_v = head >= nh + a.n_kv;
  const int g = head - nh - (is_v ? a.n_kv : 0);
  const float *row = is_q ? q + s * q_stride + (int64_t)head * hd
                          : (is_v ? v + s * v_stride : k + s * k_stride) + (int64_t)g * hd;
  uint8_t *blk = nullptr;
  if (!is_q) {
    blk = paged_block(a, paged_block_bytes(T, a.page, hd), b, p, g);
    if (!blk) return;
  }
  const int pp = (int)(p % a.page);
  for (int d = lane; d < hd; d += 64) {
    float val = row[d];
    if (!is_v && d < rd) {
      const bool first = neox ? d < half : (d & 1) == 0;
      const int i = neox ? (first ? d : d - half) : d >> 1;
      const int o = neox ? (first ? d + half : d - half) : d ^ 1;
      const float x = row[o];
      val = first ? val * cs[i] - x * sn[i] : x * sn[i] + val * cs[i];
    }
    if (is_q) {
      q_out[(s * nh + head) * (int64_t)hd + d] = val;
      continue;
    }
    const int off = is_v ? paged_v_off<T>(a.page, hd, pp, d) : paged_k_off<T>(hd, pp, d);
    if constexpr (T == kPgF16) {
      *(_Float16 *)(blk + off) = (_Float16)val;
    } else {
      int8_t n8;
      _Float16 scale;
      q8_of(val, n8, scale);
      *(int8_t *)(blk + off) = n8;
      if ((lane & 31) == 0) *(_Float16 *)(blk + (is_v ? paged_vs_off(a.page, hd, pp, d >> 5) : paged_ks_off(a.page, hd, pp, d >> 5))) = scale;
    }
  }
}

template <int T>
__global__ void __launch_bounds__(256) k_paged_read(PagedArgs a, _Float16 *__restrict__ k, _Float16 *__restrict__ v) {
  const int64_t s = blockIdx.x;
  const int b = paged_seq_of(a, s);
  if (b < 0) return;
  int64_t r0, n;
  paged_rows(a, b, r0, n);
  const int64_t p = (int64_t)a.seq_len[b] - n + (s - r0);
  const int head = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (head >= 2 * a.n_kv) return;
  const bool is_v = head >= a.n_kv;
  const int g = is_v ? head - a.n_kv : head, hd = a.hd;
  const uint8_t *blk = paged_block(a, paged_block_bytes(T, a.page, hd), b, p, g);
  const int pp = (int)(p % a.page);
  _Float16 *out = (is_v ? v : k) + (s * a.n_kv + g) * (int64_t)hd;
  for (int d = lane; d < hd; d += 64) {
    _Float16 x = 0;
    if (blk) {
      const int off = is_v ? paged_v_off<T>(a.page, hd, pp, d) : paged_k_off<T>(hd, pp, d);
      if constexpr (T == kPgF16) {
        x = *(const _Float16 *)(blk + off);
      } else {
        const int so = is_v ? paged_vs_off(a.page, hd, pp, d >> 5) : paged_ks_off(a.page, hd, pp, d >> 5);
        x = (_Float16)((float)*(const int8_t *)(blk + off) * (float)*(const _Float16 *)(blk + so));
      }
    }
    out[d] = x;
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
  for (int i = 0; i < kCopyPer; ++i)
    if (o + i * 4096 < page_bytes) x[i] = *(const uint4 *)(s + o + i * 4096);
#pragma unroll
  for (int i = 0; i < kCopyPer; ++i)
    if (o + i * 4096 < page_bytes) *(uint4 *)(d + o + i * 4096) = x[i];
}

}  // namespace

hipError_t launch_paged_store(hipStream_t st, const PagedArgs &a, const float *q, int64_t q_stride, const float *k,
                              int64_t k_stride, const float *v, int64_t v_stride, int n_head, int rope_dim,
                              const float *inv_freq, int neox, float *q_out) {
  const dim3 grid((unsigned)a.s_rows, (unsigned)((n_head + 2 * a.n_kv + 3) / 4));
  if (a.type == kPgF16)
    KMOE_LAUNCH(k_paged_store<kPgF16>, grid, dim3(256), 0, st, a, q, q_stride, k, k_stride, v, v_stride, n_head,
                rope_dim, inv_freq, neox, q_out);
  else
    KMOE_LAUNCH(k_paged_store<kPgQ8>, grid, dim3(256), 0, st, a, q, q_stride, k, k_stride, v, v_stride, n_head,
                rope_dim, inv_freq, neox, q_out);
  return hipGetLastError();
}

hipError_t launch_paged_read(hipStream_t st, const PagedArgs &a, uint16_t *k, uint16_t *v) {
  const dim3 grid((unsigned)a.s_rows, (unsigned)((2 * a.n_kv + 3) / 4));
  if (a.type == kPgF16)
    KMOE_LAUNCH(k_paged_read<kPgF16>, grid, dim3(256), 0, st, a, (_Float16 *)k, (_Float16 *)v);
  else
    KMOE_LAUNCH(k_paged_read<kPgQ8>, grid, dim3(256), 0, st, a, (_Float16 *)k, (_Float16 *)v);
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
