// kmoe_pages.hip — the host's account of a paged cache: which pages are free,
// which sequences hold which (include/kmoe.h, kmoe_pages_*). Host code only.
#include <stdint.h>
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>
#include <map>
#include <new>
#include <set>
#include <string>
#include <vector>

#include "../../include/kmoe.h"

namespace {

constexpr int64_t kMaxLen = (int64_t)1 << 30;  // what a page table spans at most (kmoe_paged_batch)

struct Seq {
  int64_t len = 0;
  std::vector<int32_t> pages;  // -1: trimmed
  int64_t window = 0;  // of the last trim that gave pages up; 0: none did
};

}  // namespace

struct kmoe_pages {
  int64_t n = 0;
  int32_t page = 0;
  std::vector<int32_t> refs;  // per page: sequences that hold it
  std::vector<int32_t> free;  // min-heap (std::greater): the lowest free page goes first
  std::map<uint32_t, Seq> seqs;
  std::string err;

  int32_t take() {
    std::pop_heap(free.begin(), free.end(), std::greater<int32_t>());
    const int32_t id = free.back();
    free.pop_back();
    refs[id] = 1;
    return id;
  }
  void give(int32_t id) {
    if (id < 0 || --refs[id] > 0) return;
    free.push_back(id);  // (reserved at creation: does not allocate)
    std::push_heap(free.begin(), free.end(), std::greater<int32_t>());
  }
};

namespace {

int pfail(kmoe_pages *p, int code, const char *fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  try {
    if (p) p->err = buf;
  } catch (...) {
  }
  return code;
}

// No exception leaves the library.
template <class F>
int guarded(kmoe_pages *p, F &&f) {
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return pfail(p, KMOE_E_BUDGET, "out of host memory");
  } catch (...) {
    return pfail(p, KMOE_E_INVALID, "unexpected error");
  }
}

// Whether s can be cut to n positions: the row that would come next sees, by the
// window, none that was trimmed, and finds the page that it goes on.
bool can_cut(const kmoe_pages *p, const Seq *s, int64_t n) {
  if (!s->window || n >= s->len) return true;
  const int64_t lo = std::max<int64_t>(0, n - s->window + 1), end = (n + p->page - 1) / p->page;
  for (int64_t i = lo / p->page; i < end; ++i)
    if (s->pages[i] < 0) return false;
  return true;
}

Seq *find(kmoe_pages *p, uint32_t seq) {
  auto it = p->seqs.find(seq);
  return it == p->seqs.end() ? nullptr : &it->second;
}

}  // namespace

extern "C" {

int kmoe_pages_create(int64_t n_pages, int32_t page, kmoe_pages **out) {
  if (!out) return KMOE_E_INVALID;
  *out = nullptr;
  if (n_pages <= 0 || n_pages > INT32_MAX || page <= 0) return KMOE_E_INVALID;
  kmoe_pages *p = nullptr;
  const int rc = guarded(nullptr, [&]() {
    p = new kmoe_pages();
    p->n = n_pages;
    p->page = page;
    p->refs.assign(n_pages, 0);
    p->free.resize(n_pages);
    for (int64_t i = 0; i < n_pages; ++i) p->free[i] = (int32_t)i;  // ascending: a min-heap
    return (int)KMOE_OK;
  });
  if (rc) {
    delete p;
    return rc;
  }
  *out = p;
  return KMOE_OK;
}

int kmoe_pages_clone(const kmoe_pages *p, kmoe_pages **out) {
  if (!out) return KMOE_E_INVALID;
  *out = nullptr;
  if (!p) return KMOE_E_INVALID;
  kmoe_pages *q = nullptr;
  const int rc = guarded(nullptr, [&]() {
    q = new kmoe_pages(*p);
    q->free.reserve(q->n);
    return (int)KMOE_OK;
  });
  if (rc) {
    delete q;
    return rc;
  }
  *out = q;
  return KMOE_OK;
}

int kmoe_pages_destroy(kmoe_pages *p) {
  delete p;
  return KMOE_OK;
}

const char *kmoe_pages_last_error(const kmoe_pages *p) { return p ? p->err.c_str() : "null pages"; }

int kmoe_pages_append_many(kmoe_pages *p, const uint32_t *seqs, const int64_t *n, int32_t count, int32_t *src,
                           int32_t *dst, int32_t *copies) {
  if (!p) return KMOE_E_INVALID;
  if (count < 0 || !copies || (count > 0 && (!seqs || !n || !src || !dst)))
    return pfail(p, KMOE_E_INVALID, "append: negative count or null pointer");
  return guarded(p, [&]() -> int {
    struct Part {
      Seq *s;
      int64_t len, want;
      bool cow;  // the new positions begin on a page that others hold too: it is copied first
    };
    *copies = 0;
    std::vector<Part> parts(count);
    std::map<uint32_t, Seq> begun;
    std::map<int32_t, int32_t> left;  // shared pages: holders that have left them so far
    std::set<uint32_t> named;
    int64_t total = 0;
    for (int32_t i = 0; i < count; ++i) {
      if (!named.insert(seqs[i]).second) return pfail(p, KMOE_E_INVALID, "append: sequence %u is named twice", seqs[i]);
      Seq *s = find(p, seqs[i]);
      const int64_t len = s ? s->len : 0, held = s ? (int64_t)s->pages.size() : 0;
      if (n[i] < 0) return pfail(p, KMOE_E_INVALID, "append: negative count");
      if (n[i] > kMaxLen - len) return pfail(p, KMOE_E_INVALID, "append: a sequence ends at %lld positions", (long long)kMaxLen);
      const int64_t want = (len + n[i] + p->page - 1) / p->page - held;
      bool cow = n[i] > 0 && len % p->page && p->refs[s->pages.back()] > 1;
      if (cow) {
        int32_t &l = left[s->pages.back()];
        cow = p->refs[s->pages.back()] - l > 1;
        l += cow;
      }
      total += want + cow;
      if (total > (int64_t)p->free.size())
        return pfail(p, KMOE_E_BUDGET, "append: %lld pages wanted, %lld free", (long long)total, (long long)p->free.size());
      if (!s) s = &begun[seqs[i]];
      s->pages.reserve(held + want);
      parts[i] = Part{s, len, want, cow};
    }
    // (from here on nothing fails)
    int32_t m = 0;
    for (int32_t i = 0; i < count; ++i) {
      const Part &t = parts[i];
      if (t.cow) {
        const int32_t old = t.s->pages.back(), id = p->take();
        --p->refs[old];
        t.s->pages.back() = id;
        src[m] = old;
        dst[m++] = id;
      }
      for (int64_t k = 0; k < t.want; ++k) t.s->pages.push_back(p->take());
      t.s->len = t.len + n[i];
    }
    p->seqs.merge(begun);
    *copies = m;
    return KMOE_OK;
  });
}

int kmoe_pages_append(kmoe_pages *p, uint32_t seq, int64_t n, int32_t *src, int32_t *dst, int32_t *copies) {
  return kmoe_pages_append_many(p, &seq, &n, 1, src, dst, copies);
}

int kmoe_pages_fork(kmoe_pages *p, uint32_t from, uint32_t to, int64_t n) {
  if (!p) return KMOE_E_INVALID;
  return guarded(p, [&]() -> int {
    Seq *s = find(p, from);
    if (!s) return pfail(p, KMOE_E_NOT_LOADED, "fork: no sequence %u", from);
    if (find(p, to)) return pfail(p, KMOE_E_INVALID, "fork: sequence %u exists", to);
    if (n < 0 || n > s->len) return pfail(p, KMOE_E_INVALID, "fork: %lld of %lld positions", (long long)n, (long long)s->len);
    if (!can_cut(p, s, n))
      return pfail(p, KMOE_E_INVALID, "fork: position %lld's window was trimmed", (long long)n);
    Seq t;
    t.len = n;
    t.window = s->window;
    t.pages.assign(s->pages.begin(), s->pages.begin() + (n + p->page - 1) / p->page);
    Seq &to_seq = p->seqs[to];
    to_seq = std::move(t);
    for (int32_t id : to_seq.pages)
      if (id >= 0) ++p->refs[id];
    return KMOE_OK;
  });
}

int kmoe_pages_truncate(kmoe_pages *p, uint32_t seq, int64_t n) {
  if (!p) return KMOE_E_INVALID;
  return guarded(p, [&]() -> int {
    Seq *s = find(p, seq);
    if (!s) return pfail(p, KMOE_E_NOT_LOADED, "truncate: no sequence %u", seq);
    if (n < 0 || n > s->len) return pfail(p, KMOE_E_INVALID, "truncate: %lld of %lld positions", (long long)n, (long long)s->len);
    if (!can_cut(p, s, n))
      return pfail(p, KMOE_E_INVALID, "truncate: position %lld's window was trimmed", (long long)n);
    const size_t keep = (size_t)((n + p->page - 1) / p->page);
    while (s->pages.size() > keep) {
      p->give(s->pages.back());
      s->pages.pop_back();
    }
    s->len = n;
    return KMOE_OK;
  });
}

int kmoe_pages_trim(kmoe_pages *p, uint32_t seq, int64_t window, int64_t n_sink, int64_t *freed) {
  if (!p) return KMOE_E_INVALID;
  return guarded(p, [&]() -> int {
    if (freed) *freed = 0;
    Seq *s = find(p, seq);
    if (!s) return pfail(p, KMOE_E_NOT_LOADED, "trim: no sequence %u", seq);
    if (window <= 0 || n_sink < 0) return pfail(p, KMOE_E_INVALID, "trim: need window > 0 and n_sink >= 0");
    // the next row sits at position len and sees p > len - window
    const int64_t lo = s->len - window + 1;
    if (lo <= 0) return KMOE_OK;
    const int64_t first = (std::min(n_sink, s->len) + p->page - 1) / p->page, last = lo / p->page;
    int64_t n = 0;
    for (int64_t i = first; i < last; ++i)
      if (s->pages[i] >= 0) {
        const bool own = p->refs[s->pages[i]] == 1;
        p->give(s->pages[i]);
        s->pages[i] = -1;
        n += own;
        s->window = window;
      }
    if (freed) *freed = n;
    return KMOE_OK;
  });
}

int kmoe_pages_drop(kmoe_pages *p, uint32_t seq) {
  if (!p) return KMOE_E_INVALID;
  return guarded(p, [&]() -> int {
    Seq *s = find(p, seq);
    if (!s) return pfail(p, KMOE_E_NOT_LOADED, "drop: no sequence %u", seq);
    for (int32_t id : s->pages) p->give(id);
    p->seqs.erase(seq);
    return KMOE_OK;
  });
}

int kmoe_pages_length(const kmoe_pages *p, uint32_t seq, int64_t *n) {
  if (!p || !n) return KMOE_E_INVALID;
  const auto it = p->seqs.find(seq);
  if (it == p->seqs.end()) return KMOE_E_NOT_LOADED;
  *n = it->second.len;
  return KMOE_OK;
}

int kmoe_pages_table(kmoe_pages *p, const uint32_t *seqs, int32_t n_seq, int32_t table_cols, int32_t *table,
                     int32_t *seq_len) {
  if (!p) return KMOE_E_INVALID;
  if (n_seq < 0 || table_cols < 0 || (n_seq > 0 && (!seqs || !seq_len || (table_cols > 0 && !table))))
    return pfail(p, KMOE_E_INVALID, "table: bad size or null pointer");
  return guarded(p, [&]() -> int {
    for (int32_t i = 0; i < n_seq; ++i) {
      Seq *s = find(p, seqs[i]);
      if (!s) return pfail(p, KMOE_E_NOT_LOADED, "table: no sequence %u", seqs[i]);
      if ((int64_t)s->pages.size() > table_cols)
        return pfail(p, KMOE_E_INVALID, "table: sequence %u holds %zu pages, %d columns", seqs[i], s->pages.size(),
                     table_cols);
    }
    for (int32_t i = 0; i < n_seq; ++i) {
      const Seq *s = find(p, seqs[i]);
      int32_t *row = table + (int64_t)i * table_cols;
      std::copy(s->pages.begin(), s->pages.end(), row);
      std::fill(row + s->pages.size(), row + table_cols, -1);
      seq_len[i] = (int32_t)s->len;
    }
    return KMOE_OK;
  });
}

int kmoe_pages_compact(kmoe_pages *p, int32_t *src, int32_t *dst, int64_t cap, int64_t *n) {
  if (!p) return KMOE_E_INVALID;
  if (cap < 0 || !n || (cap > 0 && (!src || !dst))) return pfail(p, KMOE_E_INVALID, "compact: bad size or null pointer");
  return guarded(p, [&]() -> int {
    const int64_t used = p->n - (int64_t)p->free.size();
    std::vector<int32_t> to(p->n, -1);
    std::vector<int32_t> rest;
    rest.reserve(p->n);  // its capacity holds the free list from then on
    int64_t m = 0, hole = 0;
    for (int64_t id = p->n - 1; id >= used && m < cap; --id) {
      if (!p->refs[id]) continue;
      while (p->refs[hole]) ++hole;
      src[m] = (int32_t)id;
      dst[m] = (int32_t)hole;
      to[id] = (int32_t)hole++;
      ++m;
    }
    for (int64_t i = 0; i < m; ++i) {
      p->refs[dst[i]] = p->refs[src[i]];
      p->refs[src[i]] = 0;
    }
    for (auto &kv : p->seqs)
      for (int32_t &id : kv.second.pages)
        if (id >= 0 && to[id] >= 0) id = to[id];
    for (int64_t id = 0; id < p->n; ++id)
      if (!p->refs[id]) rest.push_back((int32_t)id);  // ascending: a min-heap
    p->free.swap(rest);
    *n = m;
    return KMOE_OK;
  });
}

int kmoe_pages_usage(const kmoe_pages *p, int64_t *used, int64_t *total) {
  if (!p) return KMOE_E_INVALID;
  if (used) *used = p->n - (int64_t)p->free.size();
  if (total) *total = p->n;
  return KMOE_OK;
}

}  // extern "C"
