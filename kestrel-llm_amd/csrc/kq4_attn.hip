// kq4_attn.hip - attention over the paged int8 key/value cache (kq4_kv.h).
//
// out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j), over the keys a query sees, in one pass over the
// cache with the running maximum of a softmax. Both products run on the f16 matrix instructions: a code (8
// bits) is an f16 exactly, and each fp32 factor beside it (q, p) is a sum of two f16 (hi + lo, 21 bits and
// more), so the sums keep fp32's accuracy for two instructions instead of one. q is scaled by a power of
// two per row first, so that lo is no subnormal where it counts.
//
// S^T = K Q^T and O^T = V^T P^T: a query is a column of both, so its maximum, sum and rescaling stay in one
// lane column, and the P that the first product leaves in a lane is the second's operand as it is: a lane
// quarter (or half) owns whole groups of 16 keys, one pair of scales.
//
// With e_j = log2(p_j) + log2(vs_j) (vs_j the value scale of key j's group), O sums 2^(e_j - M) codes and l
// sums 2^(e_j - M) / vs_j, M the running maximum of e_j: the value scale costs no instruction per key, and
// the f16 range holds what O gets, whatever the scales are (they are at least 2^-100, so l stays finite).
#include "kq4_common.h"
#include "kq4_kv.h"
#include "kq4_internal.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;
constexpr float kNegInf = -__builtin_inff();
// P is held at 2^kTop for the running maximum, which is raised only where a key passes it by 2^kSlack:
// f16 holds 2^(kTop + kSlack), and lo's last bit at the maximum is 2^-31 of it.
constexpr float kTop = 6.0f, kSlack = 8.0f;

struct AttnArgs {
  kq4_kv kv;
  int log_pg;
  const float *q;
  long ldq;
  float *out;
  int heads, group;   // query heads, and those per kv head
  float scale2;       // softmax scale * log2(e)
  int window;
  int chunk, ns;      // keys per split, splits at most
  float *part_o;      // [ns][n_tok * heads][D], unnormalised
  float2 *part_ml;    // [ns][n_tok * heads] maximum, sum
};

union Frag {
  uint32_t u[4];
  half8 h;
};

// 8 codes (2 dwords of bytes, code + 128) as f16: 0x64bb is 1024 + byte, minus 1152.
KQ4_DEV half8 codes_f16(uint32_t a, uint32_t b) {
  Frag f;
  f.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
  f.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
  f.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
  f.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
  return f.h - (_Float16)1152.0f;
}

KQ4_DEV float max_xor16(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
KQ4_DEV float max_xor32(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Chunk c (16 dimensions) of a query row, rotated as the keys were (fp32 here: q is not rounded to a
// grid afterwards). cs: the row's cosines and sines, nullptr without a rotation of the row.
KQ4_DEV void load_q_chunk(const float *row, int c, int rp, const float2 *cs, bool bad, float (&x)[16]) {
#pragma unroll
  for (int e = 0; e < 16; e += 4) {
    const float4 a = *reinterpret_cast<const float4 *>(row + 16 * c + e);
    x[e] = a.x; x[e + 1] = a.y; x[e + 2] = a.z; x[e + 3] = a.w;
  }
  if (c >= 2 * rp) return;
  if (bad) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(0x7fc00000u);
    return;
  }
  const bool up = c >= rp;             // the second of a pair: x2 c + x1 s, else x1 c - x2 s
  const int o = up ? c - rp : c + rp;
  const float2 *t = cs + 16 * (up ? o : c);
#pragma unroll
  for (int e = 0; e < 16; e += 4) {
    const float4 a = *reinterpret_cast<const float4 *>(row + 16 * o + e);
    const float y[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = t[e + i];
      x[e + i] = fmaf(x[e + i], f.x, up ? y[i] * f.y : -(y[i] * f.y));
    }
  }
}

// hi + lo of 8 values at 2^sh.
KQ4_DEV void split_f16(const float *x, int sh, half8 &hi, half8 &lo) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float s = ldexpf(x[j], sh);
    hi[j] = (_Float16)s;
    lo[j] = (_Float16)(s - (float)hi[j]);
  }
}

// The exponent that brings a row's largest magnitude to [2^13, 2^14); 0 for a row of zeros.
KQ4_DEV int row_shift(float amax) {
  if (!(amax > 0.0f) || amax == __builtin_inff()) return 0;
  return 13 - ilogbf(amax);
}

// ---- up to 16 rows (query tokens * heads per kv head) a tile: decode ---------------------------------
// A workgroup is one sequence, kv head and split; its waves take 64 keys in turn straight from memory to
// registers (nothing is shared between waves until they join), the next keys' loads in flight during the
// softmax and the second product.
template <int D>
__global__ __launch_bounds__(64 * kWaves, 2) void attn_rows16_kernel(AttnArgs a) {
  constexpr int TT = D / 64, DT = D / 16, LD = D + 4;
  __shared__ float s_o[kWaves][16][LD];
  __shared__ float2 s_ml[kWaves][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i16 = lane & 15, qd = lane >> 4;
  const int seq = blockIdx.x / a.kv.kv_heads, h = blockIdx.x - seq * a.kv.kv_heads;
  const int split = blockIdx.y;
  const KQ4KvSpan sp = kq4_kv_span(a.kv.q_start[seq], a.kv.q_start[seq + 1], a.kv.kv_len[seq], a.kv.n_tok,
                                   a.kv.table_pages << (a.log_pg + 4));
  const int rows = sp.nq * a.group;
  const int *table = a.kv.block_table + (long)seq * a.kv.table_pages;
  const long n_rows = (long)a.kv.n_tok * a.heads;

  for (int r0 = 0; r0 < rows; r0 += 16) {
    const int last = r0 + 15 < rows ? r0 + 15 : rows - 1;
    int base, end;
    const int used = kq4_kv_ranges(sp, r0 / a.group, last / a.group, a.window, a.chunk, a.ns, &base, &end);
    if (split >= used) continue;
    base += split * a.chunk;
    if (split + 1 < used) end = base + a.chunk;
    const int g_end = (sp.len + 15) >> 4;      // groups that hold keys

    // this lane's query row, the keys it sees
    const int r = r0 + i16 <= last ? r0 + i16 : last;
    const int tq = r / a.group, head = h * a.group + (r - tq * a.group);
    int see_lo, see_hi;
    kq4_kv_sees(sp.p0 + tq, sp.len, a.window, &see_lo, &see_hi);
    int all_lo, all_hi, t_;                    // keys [all_lo, all_hi) every row sees
    kq4_kv_sees(sp.p0 + last / a.group, sp.len, a.window, &all_lo, &t_);
    kq4_kv_sees(sp.p0 + r0 / a.group, sp.len, a.window, &t_, &all_hi);

    half8 qh[TT][2], ql[TT][2];
    float descale;
    {
      const float *row = a.q + (sp.q0 + tq) * a.ldq + (long)head * D;
      const int rp = a.kv.rope_dim / 32;
      const float2 *cs = nullptr;
      bool bad = false;
      if (rp) {
        const int pr = a.kv.rope_pos ? a.kv.rope_pos[sp.q0 + tq] : sp.p0 + tq;
        bad = pr < 0 || pr >= a.kv.rope_rows;
        cs = reinterpret_cast<const float2 *>(a.kv.rope) + (long)(bad ? 0 : pr) * (a.kv.rope_dim / 2);
      }
      float x[TT][16], amax = 0.0f;
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        load_q_chunk(row, 4 * t + qd, rp, cs, bad, x[t]);
#pragma unroll
        for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(x[t][e]));
      }
      const int sh = row_shift(max_xor32(max_xor16(amax)));
      descale = ldexpf(a.scale2, -sh);
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) split_f16(&x[t][8 * u], sh, qh[t][u], ql[t][u]);
    }

    float4v o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = float4v{0.f, 0.f, 0.f, 0.f};
    float M = kNegInf, l = 0.0f;

    // group of this lane's key row (A operand) and of its key quarter (scales, values); -1: none
    auto group_of = [&](int key, int sub) -> long {
      const int g = (key >> 4) + sub;
      return key < end && g < g_end
                 ? kq4_kv_group_at(table, a.kv.table_pages, g, h, a.kv.n_pages, a.kv.kv_heads, a.log_pg)
                 : -1;
    };
    uint4 kr[4][TT], vr[DT];
    float2 sc = make_float2(0.f, 0.f);
    auto load_k = [&](long g) {
      const uint8_t *p = a.kv.codes + (g < 0 ? 0 : g) * (32 * D) + 256 * qd + 16 * (i16 & 3);
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
        for (int t = 0; t < TT; ++t) kr[t4][t] = *reinterpret_cast<const uint4 *>(p + 1024 * t + 64 * t4);
    };
    auto load_v = [&](long g) {
      const uint8_t *p = a.kv.codes + (g < 0 ? 0 : g) * (32 * D) + 16 * D + 16 * i16;
#pragma unroll
      for (int d = 0; d < DT; ++d) vr[d] = *reinterpret_cast<const uint4 *>(p + 256 * d);
    };

    int key = base + 64 * wave;
    long gv = group_of(key, qd);
    load_k(group_of(key, i16 >> 2));
    load_v(gv);
    if (gv >= 0) sc = *reinterpret_cast<const float2 *>(a.kv.scales + 2 * gv);
    for (; key < end; key += 64 * kWaves) {
      const int next = key + 64 * kWaves;
      const long gk_n = group_of(next, i16 >> 2), gv_n = group_of(next, qd);

      float4v s[4];
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4) {
        s[t4] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          const half8 k0 = codes_f16(kr[t4][t].x, kr[t4][t].y), k1 = codes_f16(kr[t4][t].z, kr[t4][t].w);
          s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[t][0], s[t4], 0, 0, 0);
          s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[t][0], s[t4], 0, 0, 0);
          s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[t][1], s[t4], 0, 0, 0);
          s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[t][1], s[t4], 0, 0, 0);
        }
      }
      if (next < end) load_k(gk_n);

      // this lane's 16 keys are tokens 4 t4 + r of group qd of the 64
      const bool there = gv >= 0;
      const float c = there ? sc.x * descale : 0.0f, lv = there ? __builtin_amdgcn_logf(sc.y) : 0.0f;
      const bool masked = key < all_lo || key + 64 > all_hi || __ballot(!there) != 0;
      uint32_t off = 0;   // bit 4 t4 + r: this lane's row does not see the key
      if (masked) {
        const int k0 = key + 16 * qd;
        // slots [see_lo - k0, min(see_hi, end) - k0) of the 16
        const int b = see_lo - k0, e = (see_hi < end ? see_hi : end) - k0;
        const uint32_t from = b <= 0 ? 0xffffu : b >= 16 ? 0u : 0xffffu << b;
        const uint32_t to = e <= 0 ? 0u : e >= 16 ? 0xffffu : (1u << e) - 1u;
        off = there ? ~(from & to) & 0xffffu : 0xffffu;
      }
      // (a group of which this row sees nothing may hold any scale: 0, not 0 times it)
      const float rv = there && off != 0xffffu ? __builtin_amdgcn_rcpf(sc.y) : 0.0f;
      float mx = kNegInf;
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, (off >> (4 * t4 + j)) & 1u ? kNegInf : s[t4][j]);
      float em = mx == kNegInf ? kNegInf : fmaf(mx, c, lv);
      em = max_xor32(max_xor16(em));
      if (__ballot(em > M + kSlack)) {
        const float m = em > M + kSlack ? em : M;
        const float f = M == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(M - m);
        l *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
        M = m;
      }
      const float shift = (M == kNegInf ? 0.0f : lv - M) + kTop;
      Frag ph[2], pl[2];
      float sum = 0.0f;
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          float p0 = __builtin_amdgcn_exp2f(fmaf(s[t4][j], c, shift));
          float p1 = __builtin_amdgcn_exp2f(fmaf(s[t4][j + 1], c, shift));
          if (masked) {
            p0 = (off >> (4 * t4 + j)) & 1u ? 0.0f : p0;
            p1 = (off >> (4 * t4 + j + 1)) & 1u ? 0.0f : p1;
          }
          sum += p0 + p1;
          const auto hi = __builtin_amdgcn_cvt_pkrtz(p0, p1);
          const auto lo = __builtin_amdgcn_cvt_pkrtz(p0 - (float)hi[0], p1 - (float)hi[1]);
          ph[t4 >> 1].u[2 * (t4 & 1) + (j >> 1)] = __builtin_bit_cast(uint32_t, hi);
          pl[t4 >> 1].u[2 * (t4 & 1) + (j >> 1)] = __builtin_bit_cast(uint32_t, lo);
        }
      l = fmaf(sum, rv, l);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const half8 v0 = codes_f16(vr[d].x, vr[d].y), v1 = codes_f16(vr[d].z, vr[d].w);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0].h, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0].h, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1].h, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1].h, o[d], 0, 0, 0);
      }
      if (next < end) load_v(gv_n);
      if (gv_n >= 0) sc = *reinterpret_cast<const float2 *>(a.kv.scales + 2 * gv_n);
      gv = gv_n;
    }

    // join the waves
    l = kq4_xor_add<32>(kq4_xor_add<16>(l));
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<float4v *>(&s_o[wave][i16][16 * d + 4 * qd]) = o[d];
    if (qd == 0) s_ml[wave][i16] = make_float2(M, l);
    __syncthreads();
    for (int i = threadIdx.x; i < (last - r0 + 1) * (D / 4); i += 64 * kWaves) {
      const int rr = i / (D / 4), d = 4 * (i - rr * (D / 4));
      float m = kNegInf;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_ml[w][rr].x);
      float sl = 0.0f;
      float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float2 ml = s_ml[w][rr];
        const float f = ml.x == kNegInf && ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x == kNegInf ? 0.0f : ml.x - m);
        sl = fmaf(ml.y, f, sl);
        acc += *reinterpret_cast<const float4v *>(&s_o[w][rr][d]) * f;
      }
      const int t = (r0 + rr) / a.group;
      const long row = (long)(sp.q0 + t) * a.heads + h * a.group + (r0 + rr - t * a.group);
      if (used == 1) {
        const float f = sl == 0.0f ? 0.0f : 1.0f / sl;
        *reinterpret_cast<float4v *>(a.out + row * D + d) = acc * f;
      } else {
        *reinterpret_cast<float4v *>(a.part_o + (split * n_rows + row) * D + d) = acc;
        if (d == 0) a.part_ml[split * n_rows + row] = make_float2(m, sl);
      }
    }
    __syncthreads();
  }
}

// ---- 32 rows a wave: prompts and chunks ------------------------------------------------------------
// A workgroup is NW * 32 rows (query tokens * heads per kv head) of one sequence and kv head: its waves share
// tiles of 64 keys, converted to f16 once on their way into LDS (two buffers, the next tile's loads in flight
// meanwhile). LDS holds the operands in lane order, 16 bytes a lane without bank conflicts: keys as
// [D/8][64 keys][8], values as [32-key tile][8-token half][group][D][8].
template <int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_rows32_kernel(AttnArgs a) {
  constexpr int NT = 64 * NW, TT = D / 32, DT = D / 32, NL = 8 * D / NT, TM = 32 * NW;
  constexpr int KB = D / 8 * 64 * 16, VB = 8 * D * 16;   // bytes of a tile's keys, values
  __shared__ __align__(16) uint8_t s_kv[2][KB + VB];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int i32 = lane & 31, hh = lane >> 5;
  const int h = blockIdx.x % a.kv.kv_heads, split = blockIdx.y;
  const int room = a.kv.table_pages << (a.log_pg + 4);

  // the sequence and row tile of this item, last tiles first (those of a prompt see the most keys)
  int item = (int)(gridDim.x / a.kv.kv_heads) - 1 - (int)(blockIdx.x / a.kv.kv_heads), seq = -1;
  KQ4KvSpan sp{0, 0, 0, 0};
  for (int b = 0; b < a.kv.n_seq; b += 64) {
    const int i = b + lane;
    KQ4KvSpan t{0, 0, 0, 0};
    if (i < a.kv.n_seq)
      t = kq4_kv_span(a.kv.q_start[i], a.kv.q_start[i + 1], a.kv.kv_len[i], a.kv.n_tok, room);
    const int cnt = (t.nq * a.group + TM - 1) / TM;
    int sum = cnt;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(sum, m);
      if (lane >= m) sum += o;
    }
    const unsigned long long at = __ballot(sum > item);
    if (at) {
      const int l = __ffsll((long long)at) - 1;
      item -= __builtin_amdgcn_readlane(sum - cnt, l);
      sp = KQ4KvSpan{__builtin_amdgcn_readlane(t.q0, l), __builtin_amdgcn_readlane(t.nq, l),
                     __builtin_amdgcn_readlane(t.p0, l), __builtin_amdgcn_readlane(t.len, l)};
      seq = b + l;
      break;
    }
    item -= __builtin_amdgcn_readlane(sum, 63);
  }
  if (seq < 0) return;
  const int rows = sp.nq * a.group, r0 = item * TM;
  const int last = r0 + TM - 1 < rows ? r0 + TM - 1 : rows - 1;
  int base, end;
  const int used = kq4_kv_ranges(sp, r0 / a.group, last / a.group, a.window, a.chunk, a.ns, &base, &end);
  if (split >= used) return;
  base += split * a.chunk;
  if (split + 1 < used) end = base + a.chunk;
  const int g_end = (sp.len + 15) >> 4;
  const int *table = a.kv.block_table + (long)seq * a.kv.table_pages;

  // this lane's query row; the keys that the wave's rows see, and those that all of them see
  const int w0 = r0 + 32 * wave, w1 = w0 + 31 < last ? w0 + 31 : last;
  const bool any = w0 <= last;
  const int r = w0 + i32 <= last ? w0 + i32 : last;
  const int tq = r / a.group, head = h * a.group + (r - tq * a.group);
  int see_lo, see_hi, all_lo, all_hi, wave_lo, wave_hi;
  kq4_kv_sees(sp.p0 + tq, sp.len, a.window, &see_lo, &see_hi);
  kq4_kv_sees(sp.p0 + (any ? w1 : last) / a.group, sp.len, a.window, &all_lo, &wave_hi);
  kq4_kv_sees(sp.p0 + (any ? w0 : last) / a.group, sp.len, a.window, &wave_lo, &all_hi);
  if (wave_hi > end) wave_hi = end;
  if (!any) wave_hi = 0;

  half8 qh[TT][2], ql[TT][2];
  float descale;
  {
    const float *row = a.q + (sp.q0 + tq) * a.ldq + (long)head * D;
    const int rp = a.kv.rope_dim / 32;
    const float2 *cs = nullptr;
    bool bad = false;
    if (rp) {
      const int pr = a.kv.rope_pos ? a.kv.rope_pos[sp.q0 + tq] : sp.p0 + tq;
      bad = pr < 0 || pr >= a.kv.rope_rows;
      cs = reinterpret_cast<const float2 *>(a.kv.rope) + (long)(bad ? 0 : pr) * (a.kv.rope_dim / 2);
    }
    float x[TT][16], amax = 0.0f;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      load_q_chunk(row, 2 * t + hh, rp, cs, bad, x[t]);
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(x[t][e]));
    }
    const int sh = row_shift(max_xor32(amax));
    descale = ldexpf(a.scale2, -sh);
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) split_f16(&x[t][8 * u], sh, qh[t][u], ql[t][u]);
  }

  float16v o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
  float M = kNegInf, l = 0.0f;

  auto group_of = [&](int key, int sub) -> long {
    const int g = (key >> 4) + sub;
    return key < end && g < g_end
               ? kq4_kv_group_at(table, a.kv.table_pages, g, h, a.kv.n_pages, a.kv.kv_heads, a.log_pg)
               : -1;
  };
  // load i of a thread: 16 bytes of group (64 i NW + 64 wave) / 2D, keys first; wave-uniform
  uint4 raw[NL];
  auto load = [&](int key) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int j = i * NT + 64 * wave;
      const long g = group_of(key, j / (2 * D));
      raw[i] = *reinterpret_cast<const uint4 *>(a.kv.codes + (g < 0 ? 0 : g) * (32 * D) +
                                                16 * (j % (2 * D) + lane));
    }
  };
  auto store = [&](uint8_t *buf) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int j = i * NT + 64 * wave, sub = j / (2 * D), part = j % (2 * D);
      Frag f0, f1;
      f0.h = codes_f16(raw[i].x, raw[i].y);
      f1.h = codes_f16(raw[i].z, raw[i].w);
      uint8_t *p0, *p1;
      if (part < D) {   // keys: chunk, token -> pieces 2 chunk and 2 chunk + 1, the token's lane slot
        const int c = (part + lane) >> 4, tok = lane & 15;
        const int slot = 32 * (sub >> 1) + (tok & 3) + 4 * (sub & 1) + 8 * (tok >> 2);
        p0 = buf + (2 * c * 64 + slot) * 16;
        p1 = p0 + 64 * 16;
      } else {          // values: dimension -> halves of 8 tokens
        const int d = part - D + lane;
        p0 = buf + KB + (((sub >> 1) * 4 + (sub & 1)) * D + d) * 16;
        p1 = p0 + 2 * D * 16;
      }
      *reinterpret_cast<uint4 *>(p0) = make_uint4(f0.u[0], f0.u[1], f0.u[2], f0.u[3]);
      *reinterpret_cast<uint4 *>(p1) = make_uint4(f1.u[0], f1.u[1], f1.u[2], f1.u[3]);
    }
  };

  load(base);
  int buf = 0;
  for (int key = base; key < end; key += 64, buf ^= 1) {
    store(s_kv[buf]);
    float c[2], lv[2], rv[2];
    bool there[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const long g0 = group_of(key, 2 * kt), g1 = group_of(key, 2 * kt + 1);
      const long g = hh ? g1 : g0;
      there[kt] = g >= 0;
      const float2 sc = *reinterpret_cast<const float2 *>(a.kv.scales + 2 * (g < 0 ? 0 : g));
      c[kt] = there[kt] ? sc.x * descale : 0.0f;
      lv[kt] = there[kt] ? __builtin_amdgcn_logf(sc.y) : 0.0f;
      rv[kt] = there[kt] ? __builtin_amdgcn_rcpf(sc.y) : 0.0f;
    }
    __syncthreads();
    if (key + 64 < end) load(key + 64);
    if (key >= wave_hi || key + 64 <= wave_lo) continue;   // (no barrier is left in this turn)

    const uint8_t *kb = s_kv[buf] + (hh * 2 * 64 + i32) * 16, *vb = s_kv[buf] + KB + (hh * D + i32) * 16;
    float16v s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kt][e] = 0.0f;
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const half8 k = *reinterpret_cast<const half8 *>(kb + ((4 * t + u) * 64 + 32 * kt) * 16);
          s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[t][u], s[kt], 0, 0, 0);
          s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[t][u], s[kt], 0, 0, 0);
        }
    }
    // this lane's keys: 16 of group 2 kt + hh
    const bool masked = key < all_lo || key + 64 > all_hi || __ballot(!(there[0] && there[1])) != 0;
    float em = kNegInf;
    if (masked) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int k0 = key + 32 * kt + 16 * hh;
        const int b = see_lo - k0, e = (see_hi < end ? see_hi : end) - k0;
        const uint32_t from = b <= 0 ? 0xffffu : b >= 16 ? 0u : 0xffffu << b;
        const uint32_t to = e <= 0 ? 0u : e >= 16 ? 0xffffu : (1u << e) - 1u;
        const uint32_t on = there[kt] ? from & to & 0xffffu : 0u;
        if (on == 0) c[kt] = lv[kt] = rv[kt] = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[kt][j] = (on >> j) & 1u ? s[kt][j] : kNegInf;
      }
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      float mx = s[kt][0];
#pragma unroll
      for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[kt][j]);
      em = fmaxf(em, mx == kNegInf ? kNegInf : fmaf(mx, c[kt], lv[kt]));
    }
    em = max_xor32(em);
    if (__ballot(em > M + kSlack)) {
      const float m = em > M + kSlack ? em : M;
      const float f = M == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(M - m);
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
      M = m;
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const float shift = (M == kNegInf ? 0.0f : lv[kt] - M) + kTop;
      Frag ph[2], pl[2];
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        float p0 = __builtin_amdgcn_exp2f(fmaf(s[kt][j], c[kt], shift));
        float p1 = __builtin_amdgcn_exp2f(fmaf(s[kt][j + 1], c[kt], shift));
        if (masked) {
          p0 = s[kt][j] == kNegInf ? 0.0f : p0;
          p1 = s[kt][j + 1] == kNegInf ? 0.0f : p1;
        }
        sum += p0 + p1;
        const auto hi = __builtin_amdgcn_cvt_pkrtz(p0, p1);
        const auto lo = __builtin_amdgcn_cvt_pkrtz(p0 - (float)hi[0], p1 - (float)hi[1]);
        ph[j >> 3].u[(j & 7) >> 1] = __builtin_bit_cast(uint32_t, hi);
        pl[j >> 3].u[(j & 7) >> 1] = __builtin_bit_cast(uint32_t, lo);
      }
      l = fmaf(sum, rv[kt], l);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const half8 v = *reinterpret_cast<const half8 *>(vb + ((kt * 4 + 2 * u) * D + 32 * d) * 16);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[u].h, o[d], 0, 0, 0);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[u].h, o[d], 0, 0, 0);
        }
    }
  }

  if (!any || w0 + i32 > last) return;
  l = kq4_xor_add<32>(l);
  const long row = (long)(sp.q0 + tq) * a.heads + head, n_rows = (long)a.kv.n_tok * a.heads;
  float *dst = used == 1 ? a.out + row * D : a.part_o + (split * n_rows + row) * D;
  const float f = used > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int j = 0; j < 16; j += 4)
      *reinterpret_cast<float4 *>(dst + 32 * d + 2 * j + 4 * hh) =
          make_float4(o[d][j] * f, o[d][j + 1] * f, o[d][j + 2] * f, o[d][j + 3] * f);
  if (used > 1 && hh == 0) a.part_ml[split * n_rows + row] = make_float2(M, l);
}

// Joins the splits of each row: one wave a row, 4 rows a workgroup.
template <int D>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int tile) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const long row = blockIdx.x * 4L + (threadIdx.x >> 6), n_rows = (long)a.kv.n_tok * a.heads;
  if (row >= n_rows) return;
  const int tok = (int)(row / a.heads), head = (int)(row - (long)tok * a.heads);
  KQ4KvSpan sp{0, 0, 0, 0};
  bool found = false;
  for (int b = 0; b < a.kv.n_seq && !found; b += 64) {
    const int i = b + lane;
    KQ4KvSpan t{0, 0, 0, 0};
    if (i < a.kv.n_seq)
      t = kq4_kv_span(a.kv.q_start[i], a.kv.q_start[i + 1], a.kv.kv_len[i], a.kv.n_tok,
                      a.kv.table_pages << (a.log_pg + 4));
    const unsigned long long at = __ballot(tok >= t.q0 && tok < t.q0 + t.nq);
    if (at) {
      const int l = __ffsll((long long)at) - 1;
      sp = KQ4KvSpan{__builtin_amdgcn_readlane(t.q0, l), __builtin_amdgcn_readlane(t.nq, l),
                     __builtin_amdgcn_readlane(t.p0, l), __builtin_amdgcn_readlane(t.len, l)};
      found = true;
    }
  }
  if (!found) return;   // a row behind the last sequence
  const int r = (tok - sp.q0) * a.group + head % a.group, r0 = r - r % tile;
  const int rows = sp.nq * a.group, last = r0 + tile - 1 < rows ? r0 + tile - 1 : rows - 1;
  int base, end;
  const int used = kq4_kv_ranges(sp, r0 / a.group, last / a.group, a.window, a.chunk, a.ns, &base, &end);
  if (used == 1) return;   // written by its only split
  float m = kNegInf;
  for (int s = lane; s < used; s += 64) m = fmaxf(m, a.part_ml[s * n_rows + row].x);
#pragma unroll
  for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  float sl = 0.0f, acc[E] = {};
  for (int s = 0; s < used; ++s) {
    const float2 ml = a.part_ml[s * n_rows + row];
    const float f = ml.x == kNegInf && ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x == kNegInf ? 0.0f : ml.x - m);
    sl = fmaf(ml.y, f, sl);
    const float *p = a.part_o + (s * n_rows + row) * D + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(p[e], f, acc[e]);
  }
  const float f = sl == 0.0f ? 0.0f : 1.0f / sl;
#pragma unroll
  for (int e = 0; e < E; ++e) a.out[row * D + E * lane + e] = acc[e] * f;
}

template <int D>
int launch(const AttnArgs &a, int tile, hipStream_t s) {
  constexpr int NW = 8;
  if (tile == 16) {
    attn_rows16_kernel<D><<<dim3((unsigned)a.kv.n_seq * a.kv.kv_heads, a.ns), 64 * kWaves, 0, s>>>(a);
  } else {
    const long items = (long)a.kv.n_tok * a.group / tile + a.kv.n_seq;
    attn_rows32_kernel<D, NW><<<dim3((unsigned)(items * a.kv.kv_heads), a.ns), 64 * NW, 0, s>>>(a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (a.ns > 1) {
    const long n_rows = (long)a.kv.n_tok * a.heads;
    attn_join_kernel<D><<<(unsigned)((n_rows + 3) / 4), 256, 0, s>>>(a, tile);
  }
  return (int)hipGetLastError();
}

}  // namespace

KQ4AttnPlan kq4_attn_plan(int n_tok, int n_seq, int heads, int kv_heads, int max_q, int max_kv) {
  KQ4AttnPlan p;
  const long keys = max_kv < 1 ? 1 : max_kv;
  const int group = heads / kv_heads;
  p.tile = (long)max_q * group <= 16 ? 16 : 256;
  const long step = p.tile == 16 ? 64 * kWaves : 64;           // keys of a workgroup's turn
  const long items = p.tile == 16 ? n_seq : (long)n_tok * group / p.tile + n_seq;
  const long base = items * kv_heads;                          // workgroups of one split
  const long most = (keys + step - 1) / step;
  long ns = ((p.tile == 16 ? 512 : 256) + base - 1) / base;
  if (ns > most) ns = most;
  if (ns > 1024) ns = 1024;
  if (ns < 1) ns = 1;
  p.chunk = (int)(((keys + ns - 1) / ns + step - 1) / step * step);
  p.ns = (int)((keys + p.chunk - 1) / p.chunk);
  return p;
}

int kq4_launch_attn(float *out, const kq4_kv &kv, int log_pg, const float *q, long ldq, int heads, float scale,
                    int window, const KQ4AttnPlan &plan, float *part_o, float *part_ml, hipStream_t s) {
  AttnArgs a{kv, log_pg, q, ldq, out, heads, heads / kv.kv_heads, scale * 1.44269504088896340736f, window,
             plan.chunk, plan.ns, part_o, reinterpret_cast<float2 *>(part_ml)};
  return kv.head_dim == 128 ? launch<128>(a, plan.tile, s) : launch<64>(a, plan.tile, s);
}
