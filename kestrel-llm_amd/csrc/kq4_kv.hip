// kq4_kv.hip - appending keys and values to the paged int8 cache, keys rotated on the way.
//
// One wave owns the keys, another the values, of one group (16 consecutive positions of a sequence, one kv
// head): it alone reads and writes those codes and that scale, so tokens of one call that share a group share
// its new scale without atomics, and the result does not depend on the order of waves.
//   rotated key   x1 c - x2 s, x2 c + x1 s: the products are exact in 64 bits, one rounding there and one to
//                 fp32 (so that codes next to a border do not depend on how the sum was contracted)
//   scale         s = max(s_old if the group holds earlier tokens, fl(amax / 127), 2^-100); the maximum is
//                 taken on the bit patterns, where a NaN is the largest: a group with a NaN has a NaN scale
//   codes         rint(fl(x * fl(1 / s))) + 128; where s grew, earlier codes become rint(fl(c * fl(s_old / s)))
// Keys lie as [D/16][16 tokens][16], values as [D][16 tokens], the orders in which the attention's lanes
// read 16 bytes each. A group's only new token (a decode step) is written by the byte; more of them as whole
// pieces of 16 bytes.
// Bound by memory where there is enough of it: 4096 tokens, 8 heads of 128 (44 MB in and out) 12.4 us, 3.5 TB/s (a copy
// of many times that size 4.8; here the launch and the chain of dependent loads, lengths, page, rows, are 3 us of it).
// A decode step is that chain alone: one token 2.6-3.1 us, 64 sequences 4.1. Keys and values to two waves: twice the
// loads in flight for the same chain.
#include "kq4_common.h"
#include "kq4_kv.h"
#include "kq4_internal.h"

namespace {

constexpr int kHeads = 2;   // kv heads per workgroup, two waves each

KQ4_DEV uint32_t wave_max_bits(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));    // lane xor 1
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));    // lane xor 2
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));   // rotate by 4
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));   // rotate by 8
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max((uint32_t)r[0], (uint32_t)r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)r[0], (uint32_t)r[1]);
}

KQ4_DEV uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// In the low byte: rint(q) + 128 for |q| <= 128. 1.5 * 2^23 + 128 leaves no fraction bits, so the addition rounds q
// to the nearest whole number, ties to even.
KQ4_DEV uint32_t round_byte(float q) { return __float_as_uint(q + 12583040.0f); }

KQ4_DEV uint32_t pack4(uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
  return __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u) | __builtin_amdgcn_perm(b3, b2, 0x04000c0cu);
}

// The 4 earlier codes of a dword at a larger scale.
KQ4_DEV uint32_t requant4(uint32_t w, float ratio) {
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = round_byte((float)((int)((w >> (8 * e)) & 255u) - 128) * ratio);
  return pack4(b[0], b[1], b[2], b[3]);
}
KQ4_DEV uint4 requant16(uint4 w, float ratio) {
  return make_uint4(requant4(w.x, ratio), requant4(w.y, ratio), requant4(w.z, ratio), requant4(w.w, ratio));
}

// The group's scale from its new tokens' largest bit pattern and its present one.
KQ4_DEV float group_scale(uint32_t amax_bits, float old, bool earlier) {
  uint32_t b = max(abs_bits(__uint_as_float(amax_bits) / 127.0f), __float_as_uint(0x1p-100f));
  if (earlier) b = max(b, abs_bits(old));
  return __uint_as_float(b);
}

// x1 c - x2 s and x2 c + x1 s: both products are exact in 64 bits, so each fma rounds the exact sum.
KQ4_DEV void rotate(float &x1, float &x2, float2 cs) {
  const double a = x1, b = x2, c = cs.x, s = cs.y;
  x1 = (float)__builtin_fma(a, c, -(b * s));
  x2 = (float)__builtin_fma(b, c, a * s);
}

// Row of the rotation table for the token at position pos, or -1 where the table has none.
KQ4_DEV int rope_row(const kq4_kv &kv, long token, int pos) {
  const int row = kv.rope_pos ? kv.rope_pos[token] : pos;
  return row >= 0 && row < kv.rope_rows ? row : -1;
}

// The group's slots [lo, hi) are new, slot s is row t0 + s of the call; slots below lo hold earlier tokens.
struct Group {
  int pos0, lo, hi;
  long t0;
  uint8_t *codes;   // of its keys, or of its values
  float *scale;
  float old;
};

template <int D>
KQ4_DEV void append_keys(const kq4_kv &kv, const float *__restrict__ k, long ldk, int head, const Group &g) {
  const int lane = threadIdx.x & 63, rp = kv.rope_dim / 32;
  const bool earlier = g.lo > 0;
  const float nan = __uint_as_float(0x7fc00000u);
  // several tokens, and a group whose scale grows: a lane has two chunks of 16 dimensions of one token, the two
  // that a rotation pairs
  constexpr int U = D / 32;                                        // such units of a token
  const int tok = lane / U, u = lane % U;
  const int ca = u < rp ? u : 2 * rp + 2 * (u - rp), cb = u < rp ? u + rp : ca + 1;
  uint4 *pa = reinterpret_cast<uint4 *>(g.codes + ca * 256 + tok * 16);
  uint4 *pb = reinterpret_cast<uint4 *>(g.codes + cb * 256 + tok * 16);
  float s;
  if (g.hi - g.lo == 1) {
    // one token: a lane has one pair of dimensions
    const int h = kv.rope_dim / 2;
    const int da = lane < h ? lane : 2 * lane, db = lane < h ? lane + h : da + 1;
    float a = 0.0f, b = 0.0f;
    if (lane < D / 2) {
      const float *p = k + (g.t0 + g.lo) * ldk + (long)head * D;
      a = p[da];
      b = p[db];
      if (lane < h) {
        const int row = rope_row(kv, g.t0 + g.lo, g.pos0 + g.lo);
        if (row >= 0) rotate(a, b, reinterpret_cast<const float2 *>(kv.rope)[(long)row * h + lane]);
        else a = b = nan;
      }
    }
    s = group_scale(wave_max_bits(max(abs_bits(a), abs_bits(b))), g.old, earlier);
    const float inv = s < __builtin_inff() ? 1.0f / s : 0.0f;
    if (!(s < __builtin_inff())) a = b = 0.0f;   // (codes of a scale that is no number are 0)
    if (lane < D / 2) {
      uint8_t *p = g.codes + g.lo * 16;
      p[(da >> 4) * 256 + (da & 15)] = (uint8_t)round_byte(a * inv);
      p[(db >> 4) * 256 + (db & 15)] = (uint8_t)round_byte(b * inv);
    }
  } else {
    float ka[16], kb[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) ka[e] = kb[e] = 0.0f;
    const bool mine = lane < 16 * U && tok >= g.lo && tok < g.hi;
    uint32_t m = 0;
    if (mine) {
      const float *p = k + (g.t0 + tok) * ldk + (long)head * D;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const float4 a = *reinterpret_cast<const float4 *>(p + 16 * ca + e);
        const float4 b = *reinterpret_cast<const float4 *>(p + 16 * cb + e);
        ka[e] = a.x; ka[e + 1] = a.y; ka[e + 2] = a.z; ka[e + 3] = a.w;
        kb[e] = b.x; kb[e + 1] = b.y; kb[e + 2] = b.z; kb[e + 3] = b.w;
      }
      if (u < rp) {
        const int row = rope_row(kv, g.t0 + tok, g.pos0 + tok);
        const float4 *cs = reinterpret_cast<const float4 *>(kv.rope + (long)(row < 0 ? 0 : row) * kv.rope_dim) + 8 * ca;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float4 f = cs[e / 2];
          rotate(ka[e], kb[e], make_float2(f.x, f.y));
          rotate(ka[e + 1], kb[e + 1], make_float2(f.z, f.w));
        }
        if (row < 0)
#pragma unroll
          for (int e = 0; e < 16; ++e) ka[e] = kb[e] = nan;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) m = max(m, max(abs_bits(ka[e]), abs_bits(kb[e])));
    }
    s = group_scale(wave_max_bits(m), g.old, earlier);
    const float inv = s < __builtin_inff() ? 1.0f / s : 0.0f;
    if (!(s < __builtin_inff()))
#pragma unroll
      for (int e = 0; e < 16; ++e) ka[e] = kb[e] = 0.0f;
    if (mine) {
      uint32_t a[4], b[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        a[d] = pack4(round_byte(ka[4 * d] * inv), round_byte(ka[4 * d + 1] * inv), round_byte(ka[4 * d + 2] * inv),
                     round_byte(ka[4 * d + 3] * inv));
        b[d] = pack4(round_byte(kb[4 * d] * inv), round_byte(kb[4 * d + 1] * inv), round_byte(kb[4 * d + 2] * inv),
                     round_byte(kb[4 * d + 3] * inv));
      }
      *pa = make_uint4(a[0], a[1], a[2], a[3]);
      *pb = make_uint4(b[0], b[1], b[2], b[3]);
    }
  }
  if (earlier && s > g.old && lane < 16 * U && tok < g.lo) {
    const float r = g.old / s;
    *pa = requant16(*pa, r);
    *pb = requant16(*pb, r);
  }
  if (lane == 0) *g.scale = s;
}

template <int D>
KQ4_DEV void append_values(const float *__restrict__ v, long ldv, int head, const Group &g) {
  constexpr int NV = D / 64;   // neighbouring dimensions of a lane
  const int lane = threadIdx.x & 63;
  const bool earlier = g.lo > 0;
  const float *row = v + g.t0 * ldv + (long)head * D + NV * lane;
  uint4 *p = reinterpret_cast<uint4 *>(g.codes + NV * lane * 16);
  float s;
  if (g.hi - g.lo == 1) {
    float x[NV];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x[j] = row[g.lo * ldv + j];
      m = max(m, abs_bits(x[j]));
    }
    s = group_scale(wave_max_bits(m), g.old, earlier);
    const float inv = s < __builtin_inff() ? 1.0f / s : 0.0f;
    const bool number = s < __builtin_inff();
    if (earlier && s > g.old) {   // (the new slot, and those behind it, are put back as they were)
      const float r = g.old / s;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const uint4 w = p[j];
        const uint4 q = requant16(w, r);
        const uint32_t before[4] = {w.x, w.y, w.z, w.w}, after[4] = {q.x, q.y, q.z, q.w};
        uint32_t o[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int n = g.lo - 4 * d;   // of the dword's slots, so many are earlier tokens'
          const uint32_t mask = n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1u;
          o[d] = (after[d] & mask) | (before[d] & ~mask);
        }
        p[j] = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
      reinterpret_cast<uint8_t *>(p + j)[g.lo] = (uint8_t)round_byte(number ? x[j] * inv : 0.0f);
  } else {
    float x[16][NV];
    uint32_t m = 0;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
#pragma unroll
      for (int j = 0; j < NV; ++j) x[t][j] = 0.0f;
      if (t >= g.lo && t < g.hi) {
        if constexpr (NV == 2) {
          const float2 f = *reinterpret_cast<const float2 *>(row + t * ldv);
          x[t][0] = f.x;
          x[t][1] = f.y;
        } else {
          x[t][0] = row[t * ldv];
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 16; ++t)
#pragma unroll
      for (int j = 0; j < NV; ++j) m = max(m, abs_bits(x[t][j]));
    s = group_scale(wave_max_bits(m), g.old, earlier);
    const float inv = s < __builtin_inff() ? 1.0f / s : 0.0f;
    if (!(s < __builtin_inff()))
#pragma unroll
      for (int t = 0; t < 16; ++t)
#pragma unroll
        for (int j = 0; j < NV; ++j) x[t][j] = 0.0f;
    const bool whole = g.lo == 0 && g.hi == 16, grew = earlier && s > g.old;
    const float r = grew ? g.old / s : 1.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      uint32_t n[4];
#pragma unroll
      for (int d = 0; d < 4; ++d)
        n[d] = pack4(round_byte(x[4 * d][j] * inv), round_byte(x[4 * d + 1][j] * inv), round_byte(x[4 * d + 2][j] * inv),
                     round_byte(x[4 * d + 3][j] * inv));
      if (!whole) {
        const uint4 w = p[j];
        const uint4 q = grew ? requant16(w, r) : w;
        const uint32_t before[4] = {w.x, w.y, w.z, w.w}, after[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int nl = g.lo - 4 * d, nh = g.hi - 4 * d;
          const uint32_t low = nl <= 0 ? 0u : nl >= 4 ? ~0u : (1u << (8 * nl)) - 1u;    // earlier tokens' bytes
          const uint32_t upto = nh <= 0 ? 0u : nh >= 4 ? ~0u : (1u << (8 * nh)) - 1u;   // and the new ones'
          n[d] = (after[d] & low) | (n[d] & upto & ~low) | (before[d] & ~upto);
        }
      }
      p[j] = make_uint4(n[0], n[1], n[2], n[3]);
    }
  }
  if (lane == 0) *g.scale = s;
}

template <int D>
__global__ __launch_bounds__(128 * kHeads) void kv_append_kernel(kq4_kv kv, int log_pg, const float *__restrict__ k,
                                                                 long ldk, const float *__restrict__ v, long ldv) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int head = blockIdx.y * kHeads + (wave >> 1), part = wave & 1;
  if (head >= kv.kv_heads) return;
  const int room = kv.table_pages << (log_pg + 4);

  // the sequence and group of item blockIdx.x: 64 sequences' counts at a time, prefix sums over the wave
  int item = blockIdx.x, seq = -1, grp = 0;
  KQ4KvSpan sp{0, 0, 0, 0};
  for (int b = 0; b < kv.n_seq; b += 64) {
    const int i = b + lane;
    KQ4KvSpan t{0, 0, 0, 0};
    int first = 0, cnt = 0;
    if (i < kv.n_seq) {
      t = kq4_kv_span(kv.q_start[i], kv.q_start[i + 1], kv.kv_len[i], kv.n_tok, room);
      cnt = kq4_kv_groups(t, &first);
    }
    const int sum = kq4_scan_add(cnt);
    const unsigned long long at = __ballot(sum > item);
    if (at) {
      const int l = __ffsll((long long)at) - 1;
      grp = __builtin_amdgcn_readlane(first + item - (sum - cnt), l);
      sp = KQ4KvSpan{__builtin_amdgcn_readlane(t.q0, l), __builtin_amdgcn_readlane(t.nq, l),
                     __builtin_amdgcn_readlane(t.p0, l), __builtin_amdgcn_readlane(t.len, l)};
      seq = b + l;
      break;
    }
    item -= __builtin_amdgcn_readlane(sum, 63);
  }
  if (seq < 0) return;   // more items than groups
  const long gi = kq4_kv_group_at(kv.block_table + (long)seq * kv.table_pages, kv.table_pages, grp, head,
                                  kv.n_pages, kv.kv_heads, log_pg);
  if (gi < 0) return;   // no page: nothing to write to
  Group g;
  g.pos0 = grp * 16;
  g.lo = sp.p0 > g.pos0 ? sp.p0 - g.pos0 : 0;
  g.hi = sp.len - g.pos0 < 16 ? sp.len - g.pos0 : 16;
  g.t0 = (long)sp.q0 + g.pos0 - sp.p0;
  g.codes = kv.codes + gi * (32 * D) + part * (16 * D);
  g.scale = kv.scales + 2 * gi + part;
  g.old = g.lo > 0 ? *g.scale : 0.0f;
  if (part == 0)
    append_keys<D>(kv, k, ldk, head, g);
  else
    append_values<D>(v, ldv, head, g);
}

}  // namespace

int kq4_launch_kv_append(const kq4_kv &kv, int log_pg, const float *k, long ldk, const float *v, long ldv,
                         hipStream_t s) {
  // a sequence's nq tokens touch at most nq / 16 + 2 groups, and no more than nq
  const long most = (long)kv.n_tok / 16 + 2L * kv.n_seq;
  const dim3 grid((unsigned)(most < kv.n_tok ? most : kv.n_tok), (kv.kv_heads + kHeads - 1) / kHeads);
  if (kv.head_dim == 128)
    kv_append_kernel<128><<<grid, 128 * kHeads, 0, s>>>(kv, log_pg, k, ldk, v, ldv);
  else
    kv_append_kernel<64><<<grid, 128 * kHeads, 0, s>>>(kv, log_pg, k, ldk, v, ldv);
  return (int)hipGetLastError();
}
