// kmoe_paged.h — the paged key-value cache's layout (internal).
//
// A page holds `pg` positions (a multiple of 32) of every kv head of one layer,
// one block per kv head. A block's elements lie in the order in which the
// attention kernels' matrix operands want them, so that a wave's load of an
// operand is one contiguous run of 16 bytes per lane and nothing is turned
// afterwards:
//   K  tiles of 16 positions by 32 dims: lane (kg, position) holds dims 8 kg ..
//      8 kg + 7 of its position (v_mfma_f32_16x16x32_f16's A operand, rows =
//      positions, k = dims)
//   V  tiles of 16 dims by 32 positions: lane (kg, dim) holds positions 4 kg ..
//      4 kg + 3 and 16 + 4 kg .. 16 + 4 kg + 3 of its dim (rows = dims, k =
//      positions, in the order in which the scores of two K tiles lie in the
//      lanes)
// f16 pages: K, V, two bytes an element. Q8_0 pages: one byte an element, two
// neighbouring tiles side by side (16 bytes a lane), after each of K and V one
// f16 scale per position and 32 dims, again in the operands' order:
//   K's bytes, K's scales, V's bytes, V's scales.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kmoe_paged_rows.h"

namespace kmoe {

constexpr int kPgF16 = 1, kPgQ8 = 8;  // ggml type ids

__host__ __device__ constexpr bool paged_type_ok(int t) { return t == kPgF16 || t == kPgQ8; }
// Bytes of one of K or V in a block.
__host__ __device__ constexpr int64_t paged_half_bytes(int t, int pg, int hd) {
  return t == kPgF16 ? (int64_t)pg * hd * 2 : (int64_t)pg * hd + (int64_t)pg * (hd / 32) * 2;
}
__host__ __device__ constexpr int64_t paged_block_bytes(int t, int pg, int hd) { return 2 * paged_half_bytes(t, pg, hd); }

// Byte offsets within a block: element (position p of the page, dim d) of K and
// of V, and for Q8_0 the scales of dims 32 u .. 32 u + 31.
template <int T>
__device__ __forceinline__ int paged_k_off(int hd, int p, int d) {
  if constexpr (T == kPgF16) return 2 * (((p >> 4) * (hd >> 5) + (d >> 5)) * 512 + ((d & 31) >> 3) * 128 + (p & 15) * 8 + (d & 7));
  return (p >> 4) * (16 * hd) + (d >> 6) * 1024 + ((d & 31) >> 3) * 256 + (p & 15) * 16 + ((d >> 5) & 1) * 8 + (d & 7);
}
// Place of position p in a V tile: group of four and element of the lane's eight.
__device__ __forceinline__ int paged_v_group(int p) { return (p & 15) >> 2; }
__device__ __forceinline__ int paged_v_elem(int p) { return (p & 3) + ((p >> 2) & 4); }
template <int T>
__device__ __forceinline__ int paged_v_off(int pg, int hd, int p, int d) {
  const int base = (int)paged_half_bytes(T, pg, hd), g = paged_v_group(p), j = paged_v_elem(p);
  if constexpr (T == kPgF16) return base + 2 * ((p >> 5) * (32 * hd) + (d >> 4) * 512 + g * 128 + (d & 15) * 8 + j);
  return base + (p >> 5) * (32 * hd) + (d >> 5) * 1024 + g * 256 + (d & 15) * 16 + ((d >> 4) & 1) * 8 + j;
}
__device__ __forceinline__ int paged_ks_off(int pg, int hd, int p, int u) {
  const int n = hd >> 5;
  return pg * hd + 2 * ((p >> 4) * (16 * n) + ((p & 15) >> 2) * (4 * n) + u * 4 + (p & 3));
}
__device__ __forceinline__ int paged_vs_off(int pg, int hd, int p, int u) {
  const int n = hd >> 5;
  return 2 * pg * hd + 2 * pg * n +
         2 * ((p >> 5) * (32 * n) + paged_v_group(p) * (8 * n) + u * 8 + paged_v_elem(p));
}

// One call's view of the cache and its rows (kmoe_paged_desc and
// kmoe_paged_batch, checked by the caller; what lies in device memory is
// checked by the kernels).
struct PagedArgs {
  int type, n_kv, hd, page;
  int64_t n_pages;
  uint8_t *pages;
  int n_seq, table_cols;
  int64_t s_rows;
  const int32_t *row_start, *seq_len, *table;
};

// Rows of sequence b, kept inside the call's.
__device__ __forceinline__ void paged_rows(const PagedArgs &a, int b, int64_t &r0, int64_t &n) {
  if (!a.row_start) {
    r0 = b;
    n = b < a.s_rows ? 1 : 0;
    return;
  }
  const RowRange r = row_range(a.row_start[b], a.row_start[b + 1], a.s_rows);
  r0 = r.r0;
  n = r.n;
}

// Block of kv head g in the page of sequence b's position p, or null where the
// table has none.
__device__ __forceinline__ uint8_t *paged_block(const PagedArgs &a, int64_t block_bytes, int b, int64_t p, int g) {
  const int64_t col = p / a.page;
  if (p < 0 || col >= a.table_cols) return nullptr;
  const int64_t id = a.table[(int64_t)b * a.table_cols + col];
  if (id < 0 || id >= a.n_pages) return nullptr;
  return a.pages + (id * a.n_kv + g) * block_bytes;
}

// The same without a window for sequences of one row that read each other's pages, which stay in
// the caches: sequence b is row b % rows * (n_seq / rows) + b / rows of q and out, and
// its row is left as it is where its length is negative.
hipError_t launch_paged_attention_again(hipStream_t st, const PagedArgs &a, int rows, const float *q, int n_head, float *out,
                                        float *part, uint32_t *counters);
// Sequences with pages in common (kmoe_paged_groups): group i holds sequences start[i] ..
// start[i + 1] - 1 and the first pages[i] columns of its first one's table. ml: maximum and
// sum of the weights of what the group's positions give a row's head, whose weighted mean
// stands in out; plan, lens: how what is left is shared out, for the launch that works it.
struct SharedArgs {
  const int32_t *start, *pages;
  int n_group;
  int rows;  // launch_paged_attention_again's
  float *ml;
  int64_t *plan;
  int32_t *lens;
  // whether a group is worth it, and all of them together: columns of a column tile (log 2)
  // when sequences are worked whole and when groups are; weight that is to be saved (0: always
  // worth it)
  int log_whole, log_cols;
  int64_t least;
};

hipError_t launch_paged_store(hipStream_t st, const PagedArgs &a, const float *q, int64_t q_stride, const float *k,
                              int64_t k_stride, const float *v, int64_t v_stride, int n_head, int rope_dim,
                              const float *inv_freq, int neox, float *q_out);
hipError_t launch_paged_read(hipStream_t st, const PagedArgs &a, uint16_t *k, uint16_t *v);
hipError_t launch_pages_copy(hipStream_t st, uint8_t *pages, int64_t n_layer, int64_t layer_stride,
                             int64_t page_bytes, const int32_t *src, const int32_t *dst, int64_t n);
// part: paged_part_floats() floats, counters: paged_counters() words, zero
// between calls; both of this call alone until it has run.
size_t paged_part_floats();
int paged_counters();
hipError_t launch_paged_attention(hipStream_t st, const PagedArgs &a, const float *q, int n_head, int64_t window,
                                  int64_t n_sink, float *out, float *part, uint32_t *counters);

// A choice of pages (kmoe_paged_attention_selected), for some of the rows by kv heads at a
// time: scores holds the ranks of pages that several work-groups score, counters (zero
// between calls) who has arrived, table and len the batch that is left, a
// sequence of one row per row and kv head (len -1: not a row of any sequence).
struct SelectArgs {
  PagedArgs a;
  const uint16_t *bounds;
  const float *q;
  int n_head, group, n_select, n_first;
  // of a launch of the attention: its sequence b is row b % rows, kv head b / rows where rows share
  // pages, otherwise the other way round
  int rows;
  uint64_t *scores;
  int32_t *table, *len;
  uint32_t *counters;
};
bool select_fits(int64_t table_cols, int n_kv);
int select_counters();
size_t select_ws_bytes();
hipError_t launch_paged_bounds(hipStream_t st, const PagedArgs &a, uint16_t *bounds);
hipError_t launch_paged_attention_selected(hipStream_t st, const PagedArgs &a, const uint16_t *bounds, const float *q,
                                           int n_head, int n_select, int n_first, float *out, float *part,
                                           uint32_t *counters, uint8_t *ws, uint32_t *select_counters);
// Rows by heads that ml holds, for kmoe_paged_attention_shared.
constexpr int64_t kSharedHeads = (int64_t)1 << 21;
size_t shared_ws_bytes();
hipError_t launch_paged_attention_shared(hipStream_t st, const PagedArgs &a, const int32_t *start, const int32_t *pages,
                                         int n_group, bool always, const float *q, int n_head, float *out, float *part,
                                         uint32_t *counters, uint8_t *ws);

}  // namespace kmoe
