// The index arithmetic of the paged cache (kq4_kv.h) as a host program calls it, for tests without a GPU.
#include "../../kestrel-llm_amd/csrc/kq4_kv.h"

extern "C" {

void t_span(int start, int end, int kv_len, int n_tok, int room, int *out) {
  const KQ4KvSpan s = kq4_kv_span(start, end, kv_len, n_tok, room);
  out[0] = s.q0; out[1] = s.nq; out[2] = s.p0; out[3] = s.len;
  out[5] = kq4_kv_groups(s, out + 4);
}

long t_group_at(const int *row, int table_pages, int group, int head, int n_pages, int kv_heads, int log_pg) {
  return kq4_kv_group_at(row, table_pages, group, head, n_pages, kv_heads, log_pg);
}

void t_sees(int p, int len, int window, int *out) { kq4_kv_sees(p, len, window, out, out + 1); }

int t_ranges(int nq, int p0, int len, int t0, int t1, int window, int chunk, int ns, int *out) {
  const KQ4KvSpan s{0, nq, p0, len};
  return kq4_kv_ranges(s, t0, t1, window, chunk, ns, out, out + 1);
}

int t_parts(int turns, int share, int most) { return kq4_kv_parts(turns, share, most); }

int t_part(int turns, int n, int *parts) { return kq4_kv_part(turns, n, parts); }

}
