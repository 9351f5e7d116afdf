// kq4_kv.hip - appending keys and values to the paged int8 cache, keys rotated on the way.
//
// One wave owns one group (16 consecutive positions of a sequence, one kv head): it alone reads and
// writes the group's codes and scales, so tokens of one call that share a group share its new scale
// without atomics, and the result does not depend on the order of waves.
//   rotated key   x1 c - x2 s, x2 c + x1 s: the products are exact in 64 bits, one rounding there and one to
//                 fp32 (so that codes next to a border do not depend on how the sum was contracted)
//   scale         s = max(s_old if the group holds earlier tokens, fl(amax / 127), 2^-100); the maximum is
//                 taken on the bit patterns, where a NaN is the largest: a group with a NaN has a NaN scale
//   codes         rint(fl(x * fl(1 / s))) + 128; where s grew, earlier codes become rint(fl(c * fl(s_old / s)))
// Keys lie as [D/16][16 tokens][16], values as [D][16 tokens], the orders in which the attention's lanes
// read 16 bytes each.
#include "kq4_common.h"
#include "kq4_kv.h"
#include "kq4_internal.h"

namespace {

constexpr int kWaves = 4;   // kv heads per workgroup

KQ4_DEV uint32_t wave_max_bits(uint32_t v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
  return v;
}

// A code + 128; 0 for the NaN that a NaN or infinite scale makes.
KQ4_DEV uint32_t code_byte(float x, float inv) {
  const float r = rintf(x * inv);
  return (uint32_t)((r == r ? (int)fminf(fmaxf(r, -127.0f), 127.0f) : 0) + 128);
}

// The 4 earlier codes of a dword at a larger scale.
KQ4_DEV uint32_t requant4(uint32_t w, float ratio) {
  uint32_t r = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const float c = (float)((int)((w >> (8 * b)) & 255u) - 128);
    r |= (uint32_t)((int)rintf(c * ratio) + 128) << (8 * b);
  }
  return r;
}

// One scale: of the new tokens' largest bit pattern and the earlier one's.
KQ4_DEV float group_scale(uint32_t amax_bits, float old, bool earlier) {
  const float s = __uint_as_float(amax_bits) / 127.0f;
  uint32_t b = max(__float_as_uint(s) & 0x7fffffffu, __float_as_uint(0x1p-100f));
  if (earlier) b = max(b, __float_as_uint(old) & 0x7fffffffu);
  return __uint_as_float(b);
}

template <int D>
__global__ __launch_bounds__(64 * kWaves) void kv_append_kernel(kq4_kv kv, int log_pg, const float *__restrict__ k,
                                                                long ldk, const float *__restrict__ v, long ldv) {
  const int lane = threadIdx.x & 63;
  const int head = blockIdx.y * kWaves + (threadIdx.x >> 6);
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
    int sum = cnt;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(sum, m);
      if (lane >= m) sum += o;
    }
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
  uint8_t *kc = kv.codes + gi * (32 * D), *vc = kc + 16 * D;

  const int pos0 = grp * 16;
  const int lo = sp.p0 > pos0 ? sp.p0 - pos0 : 0;                  // the new tokens' slots [lo, hi)
  const int hi = sp.len - pos0 < 16 ? sp.len - pos0 : 16;
  const long t0 = (long)sp.q0 + pos0 - sp.p0;                      // token of slot 0, where it is new
  const bool earlier = lo > 0;
  const float2 old = earlier ? *reinterpret_cast<const float2 *>(kv.scales + 2 * gi) : make_float2(0.f, 0.f);

  // values: D/64 neighbouring dimensions a lane
  constexpr int NV = D / 64;
  float vv[16][NV];
#pragma unroll
  for (int s = 0; s < 16; ++s) {
#pragma unroll
    for (int j = 0; j < NV; ++j) vv[s][j] = 0.f;
    if (s >= lo && s < hi) {
      const float *p = v + (t0 + s) * ldv + (long)head * D + NV * lane;
      if constexpr (NV == 2) {
        const float2 f = *reinterpret_cast<const float2 *>(p);
        vv[s][0] = f.x; vv[s][1] = f.y;
      } else {
        vv[s][0] = *p;
      }
    }
  }

  // keys: a lane has two chunks of 16 dimensions of one token, the two that a rotation pairs
  constexpr int U = D / 32;                                        // such units of a token
  const int tok = lane / U, u = lane % U, rp = kv.rope_dim / 32;
  const bool mine = lane < 16 * U && tok >= lo && tok < hi;
  const int ca = u < rp ? u : 2 * rp + 2 * (u - rp), cb = u < rp ? u + rp : ca + 1;
  float ka[16], kb[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) ka[e] = kb[e] = 0.f;
  if (mine) {
    const float *p = k + (t0 + tok) * ldk + (long)head * D;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float4 a = *reinterpret_cast<const float4 *>(p + 16 * ca + e);
      const float4 b = *reinterpret_cast<const float4 *>(p + 16 * cb + e);
      ka[e] = a.x; ka[e + 1] = a.y; ka[e + 2] = a.z; ka[e + 3] = a.w;
      kb[e] = b.x; kb[e + 1] = b.y; kb[e + 2] = b.z; kb[e + 3] = b.w;
    }
    if (u < rp) {
      const int row = kv.rope_pos ? kv.rope_pos[t0 + tok] : pos0 + tok;
      if (row >= 0 && row < kv.rope_rows) {
        const float2 *cs = reinterpret_cast<const float2 *>(kv.rope) + (long)row * (kv.rope_dim / 2) + 16 * ca;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 f = cs[e];
          const double a = ka[e], b = kb[e], c = f.x, s = f.y;
          ka[e] = (float)(a * c - b * s);
          kb[e] = (float)(b * c + a * s);
        }
      } else {   // a row that the table does not have: the token's key has no value
#pragma unroll
        for (int e = 0; e < 16; ++e) ka[e] = kb[e] = __uint_as_float(0x7fc00000u);
      }
    }
  }

  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e)
    mk = max(mk, max(__float_as_uint(ka[e]) & 0x7fffffffu, __float_as_uint(kb[e]) & 0x7fffffffu));
#pragma unroll
  for (int s = 0; s < 16; ++s)
#pragma unroll
    for (int j = 0; j < NV; ++j) mv = max(mv, __float_as_uint(vv[s][j]) & 0x7fffffffu);
  const float sk = group_scale(wave_max_bits(mk), old.x, earlier);
  const float sv = group_scale(wave_max_bits(mv), old.y, earlier);
  const float ik = 1.0f / sk, iv = 1.0f / sv;

  if (mine || (lane < 16 * U && tok < lo && sk > old.x)) {
    uint4 *pa = reinterpret_cast<uint4 *>(kc + ca * 256 + tok * 16);
    uint4 *pb = reinterpret_cast<uint4 *>(kc + cb * 256 + tok * 16);
    uint32_t a[4], b[4];
    if (mine) {
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        a[d] = b[d] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[d] |= code_byte(ka[4 * d + e], ik) << (8 * e);
          b[d] |= code_byte(kb[4 * d + e], ik) << (8 * e);
        }
      }
    } else {
      const float r = old.x / sk;
      const uint4 x = *pa, y = *pb;
      a[0] = requant4(x.x, r); a[1] = requant4(x.y, r); a[2] = requant4(x.z, r); a[3] = requant4(x.w, r);
      b[0] = requant4(y.x, r); b[1] = requant4(y.y, r); b[2] = requant4(y.z, r); b[3] = requant4(y.w, r);
    }
    *pa = make_uint4(a[0], a[1], a[2], a[3]);
    *pb = make_uint4(b[0], b[1], b[2], b[3]);
  }

  const bool whole = lo == 0 && hi == 16, grew = earlier && sv > old.y;
  const float rv = grew ? old.y / sv : 1.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    uint4 *p = reinterpret_cast<uint4 *>(vc + (NV * lane + j) * 16);
    uint32_t w[4] = {0, 0, 0, 0};
    if (!whole) {
      const uint4 x = *p;
      w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      uint32_t n = w[d];
      if (grew && 4 * d < lo) n = requant4(n, rv);   // (of the dword's slots only those below lo are taken)
      uint32_t o = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int s = 4 * d + e;
        const uint32_t b = s >= hi ? (w[d] >> (8 * e)) & 255u
                           : s < lo ? (n >> (8 * e)) & 255u
                                    : code_byte(vv[s][j], iv);
        o |= b << (8 * e);
      }
      w[d] = o;
    }
    *p = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (lane == 0) *reinterpret_cast<float2 *>(kv.scales + 2 * gi) = make_float2(sk, sv);
}

}  // namespace

int kq4_launch_kv_append(const kq4_kv &kv, int log_pg, const float *k, long ldk, const float *v, long ldv,
                         hipStream_t s) {
  // a sequence's nq tokens touch at most nq / 16 + 2 groups, and no more than nq
  const long most = (long)kv.n_tok / 16 + 2L * kv.n_seq;
  const dim3 grid((unsigned)(most < kv.n_tok ? most : kv.n_tok), (kv.kv_heads + kWaves - 1) / kWaves);
  if (kv.head_dim == 128)
    kv_append_kernel<128><<<grid, 64 * kWaves, 0, s>>>(kv, log_pg, k, ldk, v, ldv);
  else
    kv_append_kernel<64><<<grid, 64 * kWaves, 0, s>>>(kv, log_pg, k, ldk, v, ldv);
  return (int)hipGetLastError();
}
