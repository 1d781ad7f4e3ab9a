// The host's side of a paged cache: which slot holds which pages.  Plain C over the caller's arrays, no allocation; a call that
// returns an error has changed nothing.  Pages are given out lowest index first, in the order of the slots.  Only the last page of a
// sequence can be partly filled, and a partly filled page belongs to one sequence (fork copies it, truncate too).
#include <stdint.h>

#include <algorithm>

#include "bifrost_b200.h"
#include "paged_kv.h"

namespace {

int reject(int* info, int reason, long long a = 0, long long b = 0) {
  info[0] = reason;
  info[1] = (int)a;
  info[2] = (int)b;
  return BF_ERR_INVALID_ARGUMENT;
}

int64_t held(const bf_page_table* t, int64_t len) { return (len + t->page - 1) / t->page; }

// in range, and named once (`twice`: named again is fine): marks the slots with a new epoch
int check_slots(bf_page_table* t, const int64_t* s, int n, bool twice, int* info) {
  if (++t->epoch <= 0) {      // the marks' numbers have run out: start again
    for (int i = 0; i < t->slots; ++i) t->mark[i] = 0;
    t->epoch = 1;
  }
  for (int i = 0; i < n; ++i) {
    if (s[i] < 0 || s[i] >= t->slots) return reject(info, BF_PAGES_SLOT_RANGE);
    if (!twice && t->mark[s[i]] == t->epoch) return reject(info, BF_PAGES_SLOT_TWICE);
    t->mark[s[i]] = t->epoch;
  }
  return BF_OK;
}

int32_t* row(const bf_page_table* t, int64_t slot) { return t->table + slot * t->width; }

int32_t take(bf_page_table* t) {      // the caller knows that a page is free
  int p = t->low;
  while (t->refs[p]) ++p;
  t->refs[p] = 1;
  t->low = p + 1;
  --t->n_free;
  return p;
}

void drop(bf_page_table* t, int32_t p) {
  if (--t->refs[p] == 0) {
    ++t->n_free;
    if (p < t->low) t->low = p;
  }
}

bool bad(const bf_page_table* t, const void* list, int n, const int* info) {
  return !t || !info || n < 0 || (n > 0 && !list);
}

}  // namespace

extern "C" {

int bf_page_table_reserve(bf_page_table* t, const int64_t* slots, const int64_t* n, int count, int32_t* set, int* n_set,
                          int* info) {
  if (bad(t, slots, count, info) || (count > 0 && (!n || !set)) || !n_set) return BF_ERR_INVALID_ARGUMENT;
  int rc = check_slots(t, slots, count, false, info);
  if (rc) return rc;
  int64_t need = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t old = t->lens[slots[i]];
    if (n[i] < 0) return reject(info, BF_PAGES_NEGATIVE);
    if (n[i] > (int64_t)t->width * t->page - old) return reject(info, BF_PAGES_TOO_LONG);
    need += held(t, old + n[i]) - held(t, old);
  }
  if (need > t->n_free) return reject(info, BF_PAGES_FULL, need, t->n_free);
  int at = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t s = slots[i], old = t->lens[s];
    t->lens[s] = old + n[i];
    for (int64_t p = held(t, old); p < held(t, old + n[i]); ++p) {
      row(t, s)[p] = take(t);
      set[at++] = (int32_t)(s * t->width + p);
      set[at++] = row(t, s)[p];
    }
    set[at++] = (int32_t)((int64_t)t->slots * t->width + s);
    set[at++] = (int32_t)t->lens[s];
  }
  *n_set = at / 2;
  return BF_OK;
}

int bf_page_table_free(bf_page_table* t, const int64_t* slots, int count, int* info) {
  if (bad(t, slots, count, info)) return BF_ERR_INVALID_ARGUMENT;
  int rc = check_slots(t, slots, count, false, info);
  if (rc) return rc;
  for (int i = 0; i < count; ++i) {
    int32_t* r = row(t, slots[i]);
    const int64_t n = held(t, t->lens[slots[i]]);
    for (int64_t p = 0; p < n; ++p) {
      drop(t, r[p]);
      r[p] = -1;
    }
    t->lens[slots[i]] = 0;
  }
  return BF_OK;
}

int bf_page_table_fork(bf_page_table* t, const int64_t* src, const int64_t* dst, int count, int32_t* fork, int* info) {
  if (bad(t, src, count, info) || (count > 0 && (!dst || !fork))) return BF_ERR_INVALID_ARGUMENT;
  int rc = check_slots(t, dst, count, false, info);
  if (rc) return rc;
  const int filled = t->epoch;
  int64_t need = 0;
  for (int i = 0; i < count; ++i) {
    if (src[i] < 0 || src[i] >= t->slots) return reject(info, BF_PAGES_SLOT_RANGE);
    if (t->mark[src[i]] == filled) return reject(info, BF_PAGES_BOTH);
    if (t->lens[dst[i]] > 0) return reject(info, BF_PAGES_HELD);
    need += t->lens[src[i]] % t->page > 0;
  }
  if (need > t->n_free) return reject(info, BF_PAGES_FULL, need, t->n_free);
  for (int i = 0; i < count; ++i) {
    const int32_t* from = row(t, src[i]);
    int32_t* to = row(t, dst[i]);
    const int64_t len = t->lens[src[i]], full = len / t->page;
    for (int64_t p = 0; p < full; ++p) {
      to[p] = from[p];
      ++t->refs[to[p]];
    }
    int32_t* f = fork + 5 * (int64_t)i;
    f[0] = (int32_t)src[i];
    f[1] = (int32_t)dst[i];
    f[2] = (int32_t)len;
    f[3] = f[4] = -1;
    if (len % t->page) {
      f[3] = from[full];
      f[4] = to[full] = take(t);
    }
    t->lens[dst[i]] = len;
  }
  return BF_OK;
}

int bf_page_table_truncate(bf_page_table* t, const int64_t* slots, const int64_t* lens, int count, int32_t* fork, int* n_fork,
                           int32_t* set, int* n_set, int* info) {
  if (bad(t, slots, count, info) || (count > 0 && (!lens || !fork || !set)) || !n_fork || !n_set) return BF_ERR_INVALID_ARGUMENT;
  int rc = check_slots(t, slots, count, false, info);
  if (rc) return rc;
  for (int i = 0; i < count; ++i) {
    if (lens[i] < 0) return reject(info, BF_PAGES_NEGATIVE);
    if (lens[i] > t->lens[slots[i]]) return reject(info, BF_PAGES_LENGTHEN);
  }
  // the tails go back first; then a partly filled page that others still hold is copied, slot by slot (its last holder keeps it).
  // A dry run on the reference counts says whether there is room for the copies
  auto tails = [&](int by) {
    int64_t freed = 0;
    for (int i = 0; i < count; ++i)
      for (int64_t p = held(t, lens[i]); p < held(t, t->lens[slots[i]]); ++p) {
        int32_t& r = t->refs[row(t, slots[i])[p]];
        freed += by < 0 && r == 1;
        r += by;
      }
    return freed;
  };
  auto shared = [&](int i) -> int32_t {     // the page to copy, or -1
    if (lens[i] % t->page == 0) return -1;
    const int32_t p = row(t, slots[i])[lens[i] / t->page];
    return t->refs[p] > 1 ? p : -1;
  };
  const int64_t freed = tails(-1);
  int64_t need = 0;
  for (int i = 0; i < count; ++i) {
    const int32_t p = shared(i);
    fork[5 * (int64_t)i + 3] = p;
    if (p >= 0) {
      --t->refs[p];
      ++need;
    }
  }
  for (int i = 0; i < count; ++i)
    if (fork[5 * (int64_t)i + 3] >= 0) ++t->refs[fork[5 * (int64_t)i + 3]];
  tails(1);
  if (need > t->n_free + freed) return reject(info, BF_PAGES_FULL, need, t->n_free + freed);
  int at = 0, copies = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t s = slots[i];
    for (int64_t p = held(t, lens[i]); p < held(t, t->lens[s]); ++p) {
      drop(t, row(t, s)[p]);
      row(t, s)[p] = -1;
      set[at++] = (int32_t)(s * t->width + p);
      set[at++] = -1;
    }
    t->lens[s] = lens[i];
    set[at++] = (int32_t)((int64_t)t->slots * t->width + s);
    set[at++] = (int32_t)lens[i];
  }
  for (int i = 0; i < count; ++i) {
    const int32_t p = shared(i);
    if (p < 0) continue;
    int32_t* f = fork + 5 * (int64_t)copies++;
    const int32_t fresh = take(t);
    drop(t, p);
    row(t, slots[i])[lens[i] / t->page] = fresh;
    f[0] = f[1] = (int32_t)slots[i];
    f[2] = (int32_t)lens[i];
    f[3] = p;
    f[4] = fresh;
  }
  *n_fork = copies;
  *n_set = at / 2;
  return BF_OK;
}

size_t bf_share_words(int n) { return n > 0 ? (size_t)bfb::plan_words(n) : 0; }

// Sequences that come from one another share their first full pages: sorted by their pages, those with a page in common are neighbours, and the
// runs of pages that the same sequences share are the edges of their prefix tree (only a fork shares pages, so two sequences that have a page in common
// have all pages before it in common too).  A run that saves reading fewer than
// min_saved tokens is left to the runs behind it, or to the sequences' tails.
int bf_page_table_share(const bf_page_table* t, const int64_t* slots, int n, int min_saved, int32_t* plan, int32_t* scratch, int* info) {
  if (bad(t, slots, n, info) || n < 1 || !plan || !scratch || min_saved < 1) return BF_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < n; ++i)
    if (slots[i] < 0 || slots[i] >= t->slots) return reject(info, BF_PAGES_SLOT_RANGE);
  int32_t *s = plan + bfb::kPS_Head, *order = s + n, *place = order + n, *last = place + n, *skip = last + n, *runs = skip + n;
  int32_t *lcp = scratch, *node = lcp + n, *stack = node + 3 * (int64_t)n, *depth = stack + 2 * (int64_t)n;
  const auto full = [&](int b) { return (int)(t->lens[s[b]] / t->page); };
  const auto common = [&](int a, int b) {      // full pages that two sequences have in common
    const int32_t *x = row(t, s[a]), *y = row(t, s[b]);
    int lo = 0, hi = std::min(full(a), full(b));
    if (s[a] == s[b]) return hi;
    while (lo < hi) {
      const int m = (lo + hi + 1) >> 1;
      if (x[m - 1] == y[m - 1]) lo = m; else hi = m - 1;
    }
    return lo;
  };
  for (int i = 0; i < n; ++i) {
    s[i] = (int32_t)slots[i];
    order[i] = i;
  }
  std::sort(order, order + n, [&](int a, int b) {
    const int c = common(a, b), fa = full(a), fb = full(b);
    if (c < fa && c < fb) return row(t, s[a])[c] < row(t, s[b])[c];
    return fa != fb ? fa < fb : a < b;
  });
  for (int i = 0; i < n; ++i) {
    place[order[i]] = i;
    lcp[i] = i + 1 < n ? common(order[i], order[i + 1]) : 0;
    last[i] = -1;
    depth[i] = 0;
    skip[i] = 0;
  }
  // the tree's inner nodes (first place, places, depth in pages), children before parents
  int nodes = 0, top = 0;
  for (int i = 0; i < n; ++i) {
    int left = i;
    while (top > 0 && stack[2 * top - 1] > lcp[i]) {
      --top;
      left = stack[2 * top];
      node[3 * nodes] = left;
      node[3 * nodes + 1] = i - left + 1;
      node[3 * nodes + 2] = stack[2 * top + 1];
      ++nodes;
    }
    if (lcp[i] > 0 && (top == 0 || stack[2 * top - 1] < lcp[i])) {
      stack[2 * top] = left;
      stack[2 * top + 1] = lcp[i];
      ++top;
    }
  }
  int count = 0;
  for (int k = nodes - 1; k >= 0; --k) {
    const int first = node[3 * k], many = node[3 * k + 1], end = node[3 * k + 2], lead = order[first], from = skip[lead];
    if ((int64_t)(end - from) * t->page * (many - 1) < min_saved || depth[lead] >= bfb::kPS_Depth) continue;
    int32_t* r = runs + bfb::kPS_Run * (int64_t)count;
    r[0] = first;
    r[1] = many;
    r[2] = from;
    r[3] = end;
    r[4] = last[lead];
    r[5] = depth[lead];
    for (int i = first; i < first + many; ++i) {
      last[order[i]] = count;
      skip[order[i]] = end;
      ++depth[order[i]];
    }
    ++count;
  }
  plan[0] = count;
  plan[1] = n;
  plan[2] = plan[3] = 0;
  return BF_OK;
}

int bf_page_table_compact(bf_page_table* t, int32_t* move, int* n_move) {
  if (!t || !move || !n_move) return BF_ERR_INVALID_ARGUMENT;
  const int live = t->pages - t->n_free;
  int n = 0, hole = 0;
  for (int p = live; p < t->pages; ++p) {
    if (!t->refs[p]) continue;
    while (t->refs[hole]) ++hole;
    move[2 * n] = p;
    move[2 * n + 1] = hole;
    ++n;
    t->refs[hole] = t->refs[p];     // a hole below is marked as taken at once, so it is not found again
    t->refs[p] = 0;
  }
  // the rows: a page at or above `live` has moved, its new number by binary search in the ascending list
  if (n)
    for (int s = 0; s < t->slots; ++s) {
      int32_t* r = row(t, s);
      const int64_t pages = held(t, t->lens[s]);
      for (int64_t i = 0; i < pages; ++i) {
        if (r[i] < live) continue;
        int lo = 0, hi = n - 1;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (move[2 * mid] < r[i]) lo = mid + 1; else hi = mid;
        }
        r[i] = move[2 * lo + 1];
      }
    }
  t->low = live;
  *n_move = n;
  return BF_OK;
}

}  // extern "C"
