// kq4_kv.h - the paged int8 key/value cache: where a group lies and which keys a query sees. Plain
// integer arithmetic without device code, so host programs compile it too.
#pragma once

#include <stdint.h>

#include "../../include/kq4.h"

#ifdef __HIPCC__
#define KQ4_HD __host__ __device__ __forceinline__
#else
#define KQ4_HD inline
#endif

// Tokens q0 .. q0 + nq - 1 of the call are positions p0 .. p0 + nq - 1 of one sequence; its keys are
// positions 0 .. len - 1 (len <= the block table's room). p0 is negative where the cache is said to
// hold fewer tokens than the call brings: those tokens have no position, no key and an empty row.
struct KQ4KvSpan {
  int q0, nq, p0, len;
};

// Entries outside [0, n_tok] are taken as the nearest inside, so no index leaves the call's arrays.
KQ4_HD KQ4KvSpan kq4_kv_span(int start, int end, int kv_len, int n_tok, int room) {
  KQ4KvSpan s;
  s.q0 = start < 0 ? 0 : start > n_tok ? n_tok : start;
  const int q1 = end < s.q0 ? s.q0 : end > n_tok ? n_tok : end;
  s.nq = q1 - s.q0;
  const int l = kv_len < 0 ? 0 : kv_len;
  s.p0 = l - s.nq;
  s.len = l < room ? l : room;
  return s;
}

// Groups of 16 positions that the call's tokens of a sequence touch: the first one and how many.
KQ4_HD int kq4_kv_groups(const KQ4KvSpan &s, int *first) {
  const int lo = s.p0 < 0 ? 0 : s.p0;
  *first = lo >> 4;
  return lo < s.len && s.nq > 0 ? ((s.len - 1) >> 4) - (lo >> 4) + 1 : 0;
}

// Index of a group among the cache's groups (codes: * 32 * head_dim bytes; scales: * 2), or -1 where the
// table has no page of the cache for it. log_pg = log2(page_tokens / 16).
KQ4_HD long kq4_kv_group_at(const int *table_row, int table_pages, int group, int head, int n_pages,
                            int kv_heads, int log_pg) {
  const int slot = group >> log_pg;
  if (group < 0 || slot >= table_pages) return -1;
  const int page = table_row[slot];
  if (page < 0 || page >= n_pages) return -1;
  return ((((long)page * kv_heads + head) << log_pg) | (group & ((1 << log_pg) - 1)));
}

// Keys [lo, hi) that the query at position p sees: none before the window, none behind itself.
KQ4_HD void kq4_kv_sees(int p, int len, int window, int *lo, int *hi) {
  *hi = p + 1 < len ? p + 1 : len;
  if (*hi < 0) *hi = 0;
  *lo = window > 0 && p + 1 > window ? p + 1 - window : 0;
  if (*lo > *hi) *lo = *hi;
}

// Keys [*base, *end) that any of the queries t0 .. t1 of a sequence sees, *base rounded down to 64, and
// the key ranges of `chunk` keys (at most ns; the last one takes the rest) that hold them, at least 1.
KQ4_HD int kq4_kv_ranges(const KQ4KvSpan &s, int t0, int t1, int window, int chunk, int ns, int *base,
                         int *end) {
  int lo, hi;
  kq4_kv_sees(s.p0 + t1, s.len, window, &lo, end);
  kq4_kv_sees(s.p0 + t0, s.len, window, &lo, &hi);
  *base = lo & ~63;
  // (unsigned: keys and chunk together may pass 2^31)
  const int n = *end > *base ? (int)(((unsigned)(*end - *base) + chunk - 1u) / (unsigned)chunk) : 0;
  return n < 1 ? 1 : n > ns ? ns : n;
}

// Turns of `turn` keys that [base, end) takes.
KQ4_HD int kq4_kv_turns(int base, int end, int turn) { return end > base ? (end - base + turn - 1) / turn : 0; }

// Turns of each of about n equal parts (the last one takes fewer); *parts receives how many there are then.
KQ4_HD int kq4_kv_part(int turns, int n, int *parts) {
  const int part = n > 1 && turns > 1 ? (turns + n - 1) / n : turns < 1 ? 1 : turns;
  *parts = turns < 1 ? 1 : (turns + part - 1) / part;
  return part;
}

// Parts of a range of so many turns where a share is `share` turns: at most `most`, and none that saves the longest
// part fewer than 3 turns.
KQ4_HD int kq4_kv_parts(int turns, int share, int most) {
  int n = (turns + share - 1) / share;
  if (n > most) n = most;
  return n > 1 && turns - (turns + n - 1) / n >= 3 ? n : 1;
}
