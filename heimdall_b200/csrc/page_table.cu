// The host's side of a paged cache: which slot holds which pages.  Plain C over the caller's arrays, no allocation; a call that
// returns an error has changed nothing.  Pages are given out lowest index first, in the order of the slots.  Only the last page of a
// sequence can be partly filled, and a partly filled page belongs to one sequence (fork copies it, truncate too).
#include <stdint.h>

#include "bifrost_b200.h"

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
