// kmoe_paged_attn.hip — attention over the paged key-value cache.
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

// Grid (row, kv head): the heads of the group one after the other.
template <int T, int HD>
__global__ void __launch_bounds__(256) k_paged_attn_plain(PagedArgs a, const float *__restrict__ q, int nh,
                                                          int64_t window, int64_t n_sink, float *__restrict__ out) {
  const int64_t r = blockIdx.x;
  const int g = blockIdx.y, group = nh / a.n_kv;
  const int b = paged_seq_of(a, r);
  if (b < 0) return;
  int64_t r0, n;
  paged_rows(a, b, r0, n);
  const Visible vis = visible_of((int64_t)a.seq_len[b] - n + (r - r0), window, n_sink);
  for (int h = g * group; h < (g + 1) * group; ++h)
    plain_head<T, HD>(a, b, g, q + (r * nh + h) * HD, vis, out + (r * nh + h) * HD);
}

}  // namespace

hipError_t launch_paged_attention(hipStream_t st, const PagedArgs &a, const float *q, int n_head, int64_t window,
                                  int64_t n_sink, float *out) {
  const dim3 grid((unsigned)a.s_rows, (unsigned)a.n_kv);
#define KMOE_PAGED(T, H) KMOE_LAUNCH((k_paged_attn_plain<T, H>), grid, dim3(256), 0, st, a, q, n_head, window, n_sink, out)
  if (a.type == kPgF16) {
    if (a.hd == 64) KMOE_PAGED(kPgF16, 64);
    else KMOE_PAGED(kPgF16, 128);
  } else {
    if (a.hd == 64) KMOE_PAGED(kPgQ8, 64);
    else KMOE_PAGED(kPgQ8, 128);
  }
#undef KMOE_PAGED
  return hipGetLastError();
}

}  // namespace kmoe
