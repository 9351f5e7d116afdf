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
// the f16 range holds what O gets, whatever the scales are. A weight is at most 2^(kTop + kSlack) and a scale between
// 2^-100 and 2^121, so l is held at kLow: 2^25 keys of the least scale fit below 2^128 (2^14 without the factor), and
// a key of the largest scale at the maximum still counts 2^-126, the least normal number.
#include "kq4_common.h"
#include "kq4_kv.h"
#include "kq4_internal.h"

#include <limits.h>
#include <math.h>

#include <type_traits>

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kCus = 256;      // compute units of an MI355X
constexpr int kMinChunk = 128; // keys that a split of the 32-row form has at least
constexpr int kRowKeys = 80;   // and the weight of its keys against its partial sums (kq4_attn_plan)
constexpr long kPartRows = 1 << 18;   // rows of partial sums of the 16-row form, at most (136 MB of 128 dimensions)
constexpr int kJoinFew = 16;   // splits up to which a wave joins a row alone
constexpr float kNegInf = -__builtin_inff();
// P is held at 2^kTop for the running maximum, which is raised only where a key passes it by 2^kSlack:
// f16 holds 2^(kTop + kSlack), and lo's last bit at the maximum is 2^-31 of it.
constexpr float kTop = 6.0f, kSlack = 8.0f;
constexpr float kLow = 0x1p-11f;   // of a row's sum of weights, O is without it

struct AttnArgs {
  kq4_kv kv;
  const float *q;
  long ldq;
  float *out;
  int log_pg;
  int heads, group;   // query heads, and those per kv head
  float scale2;       // softmax scale * log2(e)
  int window;
  KQ4AttnPlan plan;
  // partial sums [splits][rows][D], unnormalised, then [splits][rows] maximum and sum (at kLow). Rows of the 16-row
  // form: [n_seq][kv_heads][plan.cap16]; of the 32-row form: [n_tok][heads].
  float *part16, *part32;
};
static_assert(sizeof(AttnArgs) <= 192, "a fourth line of arguments costs a short launch 0.25 us");

// A split's sums of a row, of n splits of so many rows.
KQ4_DEV float *part_o(float *part, long rows, long row, int split, int dim) { return part + (split * rows + row) * dim; }
KQ4_DEV float2 *part_ml(float *part, int n, long rows, long row, int split, int dim) {
  return reinterpret_cast<float2 *>(part + n * rows * dim) + split * rows + row;
}

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

// What a query row is rotated by: its row of the table, or none (rp: rotated chunk pairs).
struct QRope {
  int rp;
  bool bad;
  const float *cs;
};
KQ4_DEV QRope q_rope(const kq4_kv &kv, int token, int pos) {
  QRope r{kv.rope_dim / 32, false, nullptr};
  if (r.rp) {
    const int row = kv.rope_pos ? kv.rope_pos[token] : pos;
    r.bad = row < 0 || row >= kv.rope_rows;
    r.cs = kv.rope + (long)(r.bad ? 0 : row) * kv.rope_dim;
  }
  return r;
}

// Chunks c0, c0 + step, .. (16 dimensions each, N of them) of a query row, rotated as the keys were (in fp32 here: q
// is not rounded to a grid afterwards). A row that the table does not have is left as it is: the caller puts a NaN in.
template <int N>
KQ4_DEV void load_q(const float *row, const QRope &r, int c0, int step, float (*x)[16]) {
  float4v own[N][4];
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) own[k][e] = reinterpret_cast<const float4v *>(row + 16 * (c0 + k * step))[e];
  if (N % 2 == 0 && r.rp == step * N / 2) {
    // a whole head's rotation: chunks k and k + N / 2 are pairs, both this lane's
    constexpr int H = N > 1 ? N / 2 : 1;
    float4v cs[H][8];
#pragma unroll
    for (int k = 0; k < H; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[k][e] = reinterpret_cast<const float4v *>(r.cs)[8 * (c0 + k * step) + e];
#pragma unroll
    for (int k = 0; k < H; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float co = cs[k][e >> 1][2 * (e & 1)], si = cs[k][e >> 1][2 * (e & 1) + 1];
        const float u = own[k][e >> 2][e & 3], v = own[(k + H) % N][e >> 2][e & 3];
        x[k][e] = fmaf(u, co, -(v * si));
        x[(k + H) % N][e] = fmaf(v, co, u * si);
      }
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[k][e] = own[k][e >> 2][e & 3];
    const int c = c0 + k * step;
    if (c >= 2 * r.rp) continue;
    const bool up = c >= r.rp;   // the second of a pair: x2 c + x1 s, else x1 c - x2 s
    const int o = up ? c - r.rp : c + r.rp;
    const float4v *t = reinterpret_cast<const float4v *>(r.cs) + 8 * (up ? o : c);
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float4v y = reinterpret_cast<const float4v *>(row + 16 * o)[e >> 2], f = t[e >> 1], g = t[(e >> 1) + 1];
      const float co[4] = {f[0], f[2], g[0], g[2]}, si[4] = {f[1], f[3], g[1], g[3]};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[k][e + i] = fmaf(x[k][e + i], co[i], up ? y[i] * si[i] : -(y[i] * si[i]));
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

// Two weights as hi + lo (both rounded to nearest: an error without a sign of its own, which the row's sum, of the
// unrounded weights, would not share).
KQ4_DEV void split_pair(float p0, float p1, uint32_t &h, uint32_t &l) {
  // (not known to the compiler: p - hi as one fma that converts hi, not a conversion and a difference)
  float minus = -1.0f;
  asm("" : "+s"(minus));
  const half2v hi = __builtin_convertvector((float2v{p0, p1}), half2v);
  const half2v lo = __builtin_convertvector((float2v{fmaf((float)hi[0], minus, p0), fmaf((float)hi[1], minus, p1)}),
                                            half2v);
  h = __builtin_bit_cast(uint32_t, hi);
  l = __builtin_bit_cast(uint32_t, lo);
}

// Two of a lane's keys of a 32-key tile: their weights, summed and as the second product's operand.
KQ4_DEV void softmax_pair(const float16v &s, int j, float c, float shift, float &sum, Frag (&ph)[2],
                          Frag (&pl)[2]) {
  const float p0 = __builtin_amdgcn_exp2f(fmaf(s[j], c, shift));
  const float p1 = __builtin_amdgcn_exp2f(fmaf(s[j + 1], c, shift));
  sum += p0 + p1;
  uint32_t h, l;
  split_pair(p0, p1, h, l);
  // (no instruction: keeps the above from being moved towards its use, behind the matrix instructions it stands
  // between)
  asm volatile("" : "+v"(h), "+v"(l), "+v"(sum));
  ph[j >> 3].u[(j & 7) >> 1] = h;
  pl[j >> 3].u[(j & 7) >> 1] = l;
}

// Rows that have partial sums in the 16-row form.
KQ4_HD long slots_of(const AttnArgs &a) { return (long)a.kv.n_seq * a.kv.kv_heads * a.plan.cap16; }

// 2^d, d <= 0, as two factors: a row's sum over small value scales is large, and something of it is left where 2^d
// alone is 0.
KQ4_DEV float2 two_factors(float d) {
  const float a = fmaxf(d, -120.0f);
  return make_float2(__builtin_amdgcn_exp2f(a), __builtin_amdgcn_exp2f(d - a));
}

// The factors of a split's, or wave's, sums in the joined row (one without a maximum has zeros, or NaN: it keeps them).
KQ4_DEV float2 split_factors(float2 ml, float m) {
  return ml.x == kNegInf ? make_float2(1.0f, 1.0f) : two_factors(ml.x - m);
}

// ---- up to 16 rows (query tokens * heads per kv head) a tile: decode ---------------------------------
// A workgroup is one sequence, kv head and split; its waves take 64 keys in turn straight from memory to
// registers (nothing is shared between waves until they join), the next keys' loads in flight during the
// softmax and the second product. Each key is read once, without a place in the caches: 32 sequences of 8192 keys, 8 kv
// heads of 128 (537 MB) 84.7 us in whole sequences, 6.35 TB/s; of 1621 to 8192 keys (321 MB) 54.5 us, 5.9 TB/s, in
// halves by length and 4.7 us for the join; 1.01 times the bytes it owes. One of 131072 keys, 4 kv heads (134 MB) 25.2
// us and 4.5 us for the join. Bound by memory; a short call by its chain of dependent loads (lengths, page, keys) and
// the join: one token over 1001 keys 6.8 us and 3.7 us.

// How sequences are dealt to the workgroups of the 16-row form (kq4_attn_plan). kOrder, kHalves: by length; of two
// workgroups that share a CU (it takes them in order, a round of kCus and then another) one is long where the other is
// short. kHalves: the first range of the rank-th longest, the second one of the rank-th shortest. kOrder: whole
// sequences, those of the second round shortest first, the others as slots free. kShares: each sequence in as many
// ranges as its part of all keys of the batch.
enum { kPlain = 0, kOrder = 1, kHalves = 2, kShares = 3 };
KQ4_HD int kq4_attn_shares(int kv_heads, int n_seq) { return kCus / kv_heads - n_seq / 2; }
KQ4_DEV int rank_at(const AttnArgs &a, int place, int split) {
  if (a.plan.deal16 == kHalves) return split ? a.kv.n_seq - 1 - place : place;
  const int round = kCus / a.kv.kv_heads;
  return place < round ? place : place < 2 * round ? a.kv.n_seq - 1 - (place - round) : place - round;
}
// Turns that sequence i's whole range takes, 0 where it is not split (no rows, or more than its partial sums' room).
KQ4_DEV int turns_of(const AttnArgs &a, int i) {
  if (i >= a.kv.n_seq) return 0;
  const KQ4KvSpan s = kq4_kv_span(a.kv.q_start[i], a.kv.q_start[i + 1], a.kv.kv_len[i], a.kv.n_tok,
                                  a.kv.table_pages << (a.log_pg + 4));
  int base, end;
  kq4_kv_ranges(s, 0, s.nq - 1, a.window, 64, 1, &base, &end);
  return s.nq && s.nq * a.group <= a.plan.cap16 ? kq4_kv_turns(base, end, 64 * a.plan.waves16) : 0;
}
// Turns of a share: all keys of the batch over the workgroups of a kv head that have a CU each, less the half ranges
// that rounding up to whole ranges adds.
KQ4_DEV int share_turns(const AttnArgs &a, int lane) {
  int all = 0;
  for (int b = 0; b < a.kv.n_seq; b += 64) all += __builtin_amdgcn_readlane(kq4_scan_add(turns_of(a, b + lane)), 63);
  const int shares = kq4_attn_shares(a.kv.kv_heads, a.kv.n_seq);
  return all > shares ? (all + shares - 1) / shares : 1;
}
// The sequence and range of item `item` of a kv head's; false where there is none. (A tile of a sequence has no more
// ranges than its whole range.)
KQ4_DEV bool shared_item(const AttnArgs &a, int item, int share, int lane, int *seq, int *split) {
  for (int b = 0; b < a.kv.n_seq; b += 64) {
    const int n = b + lane < a.kv.n_seq ? kq4_kv_parts(turns_of(a, b + lane), share, a.plan.ns16) : 0;
    const int sum = kq4_scan_add(n);
    const unsigned long long at = __ballot(sum > item);
    if (at) {
      const int l = __ffsll((long long)at) - 1;
      *seq = b + l;
      *split = item - __builtin_amdgcn_readlane(sum - n, l);
      return true;
    }
    item -= __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}
// Keys of a range of a dealt sequence's [base, end), and how many ranges it has.
KQ4_DEV int dealt_part(const AttnArgs &a, int base, int end, int share, int *used) {
  const int turn = 64 * a.plan.waves16, turns = kq4_kv_turns(base, end, turn);
  return turn * kq4_kv_part(turns, a.plan.deal16 == kHalves ? 2 : kq4_kv_parts(turns, share, a.plan.ns16), used);
}
// The sequence with `rank` longer ones (ties by number); n_seq <= 64 NW.
template <int NW>
KQ4_DEV int ranked(const AttnArgs &a, int rank, uint8_t *lds) {
  int *s_len = reinterpret_cast<int *>(lds), *s_seq = s_len + 64 * NW;
  const int i = threadIdx.x, n = a.kv.n_seq;
  const int len = i < n ? a.kv.kv_len[i] : INT_MIN;
  s_len[i] = len;
  __syncthreads();
  int longer = 0;
  for (int j = 0; j < n; j += 4) {   // (those past n are the shortest)
    const int4 l = *reinterpret_cast<const int4 *>(s_len + j);
    longer += (l.x > len || (l.x == len && j < i)) + (l.y > len || (l.y == len && j + 1 < i)) +
              (l.z > len || (l.z == len && j + 2 < i)) + (l.w > len || (l.w == len && j + 3 < i));
  }
  if (i < n && longer == rank) *s_seq = i;
  __syncthreads();
  const int seq = __builtin_amdgcn_readfirstlane(*s_seq);
  __syncthreads();   // (the memory is used again)
  return seq;
}

template <int D, int NW>
constexpr int kLds16 = NW * 16 * ((D + 4) * 4 + 8);
template <int D, int NW>
KQ4_DEV void attn_rows16(const AttnArgs &a, int block, int split, uint8_t *lds) {
  constexpr int TT = D / 64, DT = D / 16, LD = D + 4;
  float(*s_o)[16][LD] = reinterpret_cast<float(*)[16][LD]>(lds);
  float2(*s_ml)[16] = reinterpret_cast<float2(*)[16]>(lds + NW * 16 * LD * 4);
  const int chunk = a.plan.chunk16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i16 = lane & 15, qd = lane >> 4;
  const int place = block / a.kv.kv_heads, h = block - place * a.kv.kv_heads;
  int seq = place, share = 0;
  if (a.plan.deal16 == kShares) {
    share = share_turns(a, lane);
    if (!shared_item(a, place, share, lane, &seq, &split)) return;
  } else if (a.plan.deal16 != kPlain) {
    seq = ranked<NW>(a, rank_at(a, place, split), lds);
  }
  const KQ4KvSpan sp = kq4_kv_span(a.kv.q_start[seq], a.kv.q_start[seq + 1], a.kv.kv_len[seq], a.kv.n_tok,
                                   a.kv.table_pages << (a.log_pg + 4));
  const int rows = sp.nq * a.group;
  if (rows > a.plan.max16) return;
  const bool whole = rows > a.plan.cap16;
  const int *table = a.kv.block_table + (long)seq * a.kv.table_pages;

  for (int r0 = 0; r0 < rows; r0 += 16) {
    const int last = r0 + 15 < rows ? r0 + 15 : rows - 1;
    int base, end;
    int part = chunk, used = kq4_kv_ranges(sp, r0 / a.group, last / a.group, a.window, chunk, whole ? 1 : a.plan.ns16,
                                           &base, &end);
    if (a.plan.deal16 >= kHalves && !whole) part = dealt_part(a, base, end, share, &used);
    if (split >= used) continue;
    base += split * part;
    if (split + 1 < used) end = base + part;
    const int g_end = (sp.len + 15) >> 4;      // groups that hold keys

    // this lane's query row, the keys it sees
    const int r = r0 + i16 <= last ? r0 + i16 : last;
    const int tq = r / a.group, head = h * a.group + (r - tq * a.group);
    int see_lo, see_hi;
    kq4_kv_sees(sp.p0 + tq, sp.len, a.window, &see_lo, &see_hi);
    int all_lo, all_hi, t_;                    // keys [all_lo, all_hi) every row sees
    kq4_kv_sees(sp.p0 + last / a.group, sp.len, a.window, &all_lo, &t_);
    kq4_kv_sees(sp.p0 + r0 / a.group, sp.len, a.window, &t_, &all_hi);

    float4v o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = float4v{0.f, 0.f, 0.f, 0.f};
    float M = kNegInf, l = 0.0f;

    // A step is 64 keys. Table entries are read two steps ahead, scales one; a register of keys or values is loaded
    // again for the next step as soon as its codes are converted, so both are in flight for most of a step.
    auto page_of = [&](int key, int sub) {   // of a lane's group among the step's 4; -1: none
      const int g = (key >> 4) + sub, slot = g >> a.log_pg;
      return key < end && g < g_end && slot < a.kv.table_pages ? table[slot] : -1;
    };
    auto group_of = [&](int page, int key, int sub) -> long {
      const int g = (key >> 4) + sub;
      return (unsigned)page < (unsigned)a.kv.n_pages
                 ? (((long)page * a.kv.kv_heads + h) << a.log_pg) | (g & ((1 << a.log_pg) - 1))
                 : -1;
    };
    constexpr int kStep = 64 * NW;
    const int ik = i16 >> 2;                 // this lane's key row's group; qd: that of its scales and values
    uint4 kr[4][TT], vr[DT];
    int key = base + 64 * wave;
    int page_k = page_of(key, ik), page_v = page_of(key, qd);
    int next_k = page_of(key + kStep, ik), next_v = page_of(key + kStep, qd);
    const uint8_t *kp, *vp;
    auto point = [&](long gk, long gv) {
      kp = a.kv.codes + (gk < 0 ? 0 : gk) * (32 * D) + 256 * qd + 16 * (i16 & 3);
      vp = a.kv.codes + (gv < 0 ? 0 : gv) * (32 * D) + 16 * D + 16 * i16;
    };
    long gv = group_of(page_v, key, qd);
    point(group_of(page_k, key, ik), gv);
    float2 sc = *reinterpret_cast<const float2 *>(a.kv.scales + 2 * (gv < 0 ? 0 : gv));
    if (key < end) {
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
        for (int t = 0; t < TT; ++t) kr[t4][t] = kq4_ld_nt(kp + 1024 * t + 64 * t4);
#pragma unroll
      for (int d = 0; d < DT; ++d) vr[d] = kq4_ld_nt(vp + 256 * d);
    }

    half8 qh[TT][2], ql[TT][2];
    int sh;
    {
      float x[TT][16], amax = 0.0f;
      const QRope rope = q_rope(a.kv, sp.q0 + tq, sp.p0 + tq);
      load_q<TT>(a.q + (sp.q0 + tq) * a.ldq + (long)head * D, rope, qd, 4, x);
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(x[t][e]));
      sh = row_shift(max_xor32(max_xor16(amax)));
      if (rope.bad) x[0][0] = __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) split_f16(&x[t][8 * u], sh, qh[t][u], ql[t][u]);
    }

    auto step = [&](auto more) {
      const int next = key + kStep;
      const bool there = gv >= 0;
      const float2 scale = sc;
      long gv_n = -1;
      int page_k2 = -1, page_v2 = -1;
      if constexpr (more.value) {
        page_k2 = page_of(next + kStep, ik);
        page_v2 = page_of(next + kStep, qd);
        gv_n = group_of(next_v, next, qd);
        point(group_of(next_k, next, ik), gv_n);
        sc = *reinterpret_cast<const float2 *>(a.kv.scales + 2 * (gv_n < 0 ? 0 : gv_n));
      }
      float4v s[4];
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4) {
        s[t4] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          const half8 k0 = codes_f16(kr[t4][t].x, kr[t4][t].y), k1 = codes_f16(kr[t4][t].z, kr[t4][t].w);
          if constexpr (more.value) kr[t4][t] = kq4_ld_nt(kp + 1024 * t + 64 * t4);
          s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[t][0], s[t4], 0, 0, 0);
          s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[t][0], s[t4], 0, 0, 0);
          s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[t][1], s[t4], 0, 0, 0);
          s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[t][1], s[t4], 0, 0, 0);
        }
      }

      // this lane's 16 keys are tokens 4 t4 + j of group qd of the 64
      // (2^-sh last: alone with scale2 it is subnormal for queries below 2^-110)
      float c = there ? ldexpf(scale.x * a.scale2, -sh) : 0.0f, lv = there ? __builtin_amdgcn_logf(scale.y) : 0.0f;
      float rv = there ? __builtin_amdgcn_rcpf(scale.y) : 0.0f;
      const bool masked = key < all_lo || key + 64 > all_hi || __ballot(!there) != 0;
      if (masked) {
        const int k0 = key + 16 * qd;
        // slots [see_lo - k0, min(see_hi, end) - k0) of the 16
        const int b = see_lo - k0, e = (see_hi < end ? see_hi : end) - k0;
        const uint32_t from = b <= 0 ? 0xffffu : b >= 16 ? 0u : 0xffffu << b;
        const uint32_t to = e <= 0 ? 0u : e >= 16 ? 0xffffu : (1u << e) - 1u;
        const uint32_t on = there ? from & to & 0xffffu : 0u;
        // (a group of which this row sees nothing may hold any scale: 0, not 0 times it)
        if (on == 0) c = lv = rv = 0.0f;
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[t4][j] = (on >> (4 * t4 + j)) & 1u ? s[t4][j] : kNegInf;
      }
      float mx = s[0][0];
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[t4][j]);
      float em = mx == kNegInf ? kNegInf : fmaf(mx, c, lv);
      em = max_xor32(max_xor16(em));
      if (__ballot(em > M + kSlack)) {
        const float m = em > M + kSlack ? em : M;
        const float2 by = two_factors(M == kNegInf ? kNegInf : M - m);
        const float f = by.x * by.y;
        l = l * by.y * by.x;
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
            p0 = s[t4][j] == kNegInf ? 0.0f : p0;
            p1 = s[t4][j + 1] == kNegInf ? 0.0f : p1;
          }
          sum += p0 + p1;
          split_pair(p0, p1, ph[t4 >> 1].u[2 * (t4 & 1) + (j >> 1)], pl[t4 >> 1].u[2 * (t4 & 1) + (j >> 1)]);
        }
      l = fmaf(sum * kLow, rv, l);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const half8 v0 = codes_f16(vr[d].x, vr[d].y), v1 = codes_f16(vr[d].z, vr[d].w);
        if constexpr (more.value) vr[d] = kq4_ld_nt(vp + 256 * d);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0].h, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0].h, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1].h, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1].h, o[d], 0, 0, 0);
      }
      key = next;
      gv = gv_n;
      next_k = page_k2;
      next_v = page_v2;
    };
    while (key + kStep < end) step(std::true_type{});
    if (key < end) step(std::false_type{});

    // join the waves
    l = kq4_xor_add<32>(kq4_xor_add<16>(l));
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<float4v *>(&s_o[wave][i16][16 * d + 4 * qd]) = o[d];
    if (qd == 0) s_ml[wave][i16] = make_float2(M, l);
    __syncthreads();
    for (int i = threadIdx.x; i < (last - r0 + 1) * (D / 4); i += 64 * NW) {
      const int rr = i / (D / 4), d = 4 * (i - rr * (D / 4));
      float m = kNegInf;
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, s_ml[w][rr].x);
      float sl = 0.0f;
      float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float2 ml = s_ml[w][rr];
        const float2 f = split_factors(ml, m);
        sl = fmaf(ml.y * f.y, f.x, sl);
        acc += *reinterpret_cast<const float4v *>(&s_o[w][rr][d]) * (f.x * f.y);
      }
      if (used == 1) {
        const int t = (r0 + rr) / a.group;
        const long row = (long)(sp.q0 + t) * a.heads + h * a.group + (r0 + rr - t * a.group);
        const float f = sl == 0.0f ? 0.0f : 1.0f / sl;
        *reinterpret_cast<float4v *>(a.out + row * D + d) = (acc * kLow) * f;
      } else {
        const int slot = (seq * a.kv.kv_heads + h) * a.plan.cap16 + r0 + rr;
        *reinterpret_cast<float4v *>(part_o(a.part16, slots_of(a), slot, split, D) + d) = acc;
        if (d == 0) *part_ml(a.part16, a.plan.ns16, slots_of(a), slot, split, D) = make_float2(m, sl);
      }
    }
    __syncthreads();
  }
}

// ---- 32 rows a wave: prompts and chunks ------------------------------------------------------------
// A workgroup is NW * 32 rows (query tokens * heads per kv head) of one sequence and kv head: its waves share
// tiles of 32 keys, converted to f16 once on their way into a ring of 4 in LDS, the loads of the tile after next
// in flight meanwhile. LDS holds the operands in lane order, 16 bytes a lane without bank conflicts: keys as
// [D/8][32 keys][8], values as [8-token half][group][D][8]. The scores of tile n + 1 are formed while tile n's go
// through the softmax, so matrix instructions and vector instructions of a wave are independent of each other.
// A prompt of 4096 tokens, 32 heads, 8 kv heads of 128: 250 us, 550 TFLOP/s of the definition's 137 GFLOP, twice that
// of matrix instructions (hi + lo). Bound by issue: a tile and wave has 32 matrix instructions (1024 cycles of its
// SIMD) and about 130 vector instructions (712, 16 of them exponentials), 1930 cycles are measured; the matrix unit
// is busy 53 % of the cycles at 1.93 GHz. A call of one tile takes 6.8 us at 64 dimensions, 9.5 at 128 (dependent
// loads, the rotation of the queries); a further tile of 4 waves 0.7 and 0.95 us.
template <int D>
constexpr int kLds32 = 4 * 64 * D * 2 + 64;
template <int D, int NW>
KQ4_DEV void attn_rows32(const AttnArgs &a, int block, int blocks, int split, uint8_t *lds) {
  constexpr int NT = 64 * NW, TT = D / 32, DT = D / 32, TM = 32 * NW;
  constexpr int L = 4 * D, NL = (L + NT - 1) / NT;      // 16-byte loads of a tile, of a thread
  constexpr int KB = D / 8 * 32 * 16;                   // bytes of a tile's keys in LDS, and of its values
  uint8_t(*s_kv)[2 * KB] = reinterpret_cast<uint8_t(*)[2 * KB]>(lds);
  float2v(*s_sc)[2] = reinterpret_cast<float2v(*)[2]>(lds + 8 * KB);
  const int chunk = a.plan.chunk32, ns = a.plan.ns32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int i32 = lane & 31, hh = lane >> 5;
  const int h = block % a.kv.kv_heads;
  const int room = a.kv.table_pages << (a.log_pg + 4);

  // the sequence and row tile of this item, last tiles first (those of a prompt see the most keys)
  int item = blocks / a.kv.kv_heads - 1 - block / a.kv.kv_heads, seq = -1;
  KQ4KvSpan sp{0, 0, 0, 0};
  for (int b = 0; b < a.kv.n_seq; b += 64) {
    const int i = b + lane;
    KQ4KvSpan t{0, 0, 0, 0};
    if (i < a.kv.n_seq)
      t = kq4_kv_span(a.kv.q_start[i], a.kv.q_start[i + 1], a.kv.kv_len[i], a.kv.n_tok, room);
    const int cnt = t.nq * a.group > a.plan.max16 ? (t.nq * a.group + TM - 1) / TM : 0;
    const int sum = kq4_scan_add(cnt);
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
  const int used = kq4_kv_ranges(sp, r0 / a.group, last / a.group, a.window, chunk, ns, &base, &end);
  if (split >= used) return;
  base += split * chunk;
  if (split + 1 < used) end = base + chunk;
  const int g_end = (sp.len + 15) >> 4;
  const int *table = a.kv.block_table + (long)seq * a.kv.table_pages;

  // this lane's query row; the keys it sees, and those that all of the wave's rows see
  const int w0 = r0 + 32 * wave, w1 = w0 + 31 < last ? w0 + 31 : last;
  const bool any = w0 <= last;
  const int r = w0 + i32 <= last ? w0 + i32 : last;
  const int tq = r / a.group, head = h * a.group + (r - tq * a.group);
  int see_lo, see_hi, all_lo, all_hi, t_;
  kq4_kv_sees(sp.p0 + tq, sp.len, a.window, &see_lo, &see_hi);
  kq4_kv_sees(sp.p0 + (any ? w1 : last) / a.group, sp.len, a.window, &all_lo, &t_);
  kq4_kv_sees(sp.p0 + (any ? w0 : last) / a.group, sp.len, a.window, &t_, &all_hi);
  if (see_hi > end) see_hi = end;

  float16v o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
  float M = kNegInf, l = 0.0f;

  // Table entries are read a tile before the loads that they lead to, one per half of the wave; those loads a
  // tile before they go to LDS, there a tile before use. A thread's load i is 16 bytes of group
  // (i NT + 64 wave) / 2D of the tile, keys first.
  const int tiles = (end - base + 31) >> 5;
  auto entry = [&](int n) {
    const int slot = (((base + 32 * n) >> 4) + hh) >> a.log_pg;
    return table[slot < a.kv.table_pages ? slot : a.kv.table_pages - 1];
  };
  // Index of a tile's group among the cache's, and whether it holds keys; without a branch, so that the loads stand
  // among the matrix instructions (where there is none: a group of page 0, never used)
  auto group_of = [&](int n, int half, int page, bool &ok) -> long {
    const int g = ((base + 32 * n) >> 4) + half;   // (g < g_end: the table has an entry for it)
    ok = (g < g_end) & ((unsigned)page < (unsigned)a.kv.n_pages);
    return (((long)(page & -(int)ok) * a.kv.kv_heads + h) << a.log_pg) | (g & ((1 << a.log_pg) - 1));
  };
  uint4v raw[NL];
  float2v raw_sc = {1.0f, 0.0f};
  bool raw_there = false;
  int ent, put0[NL], put1[NL];   // table entries of the tile after raw's; where a load's halves go in LDS
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int j = i * NT + 64 * wave, half = j / (2 * D), part = j % (2 * D);
    if (part < D) {   // keys: chunk, token -> pieces 2 chunk and 2 chunk + 1, the token's lane slot
      const int c = (part + lane) >> 4, tok = lane & 15;
      put0[i] = (2 * c * 32 + (tok & 3) + 4 * half + 8 * (tok >> 2)) * 16;
      put1[i] = put0[i] + 32 * 16;
    } else {          // values: dimension -> halves of 8 tokens
      put0[i] = KB + (half * D + part - D + lane) * 16;
      put1[i] = put0[i] + 2 * D * 16;
    }
  }
  auto fetch_tile = [&](int n, int entries, uint4v (&kv)[NL], float2v &sc, bool &there) {
    bool ok0, ok1;
    const long g0 = group_of(n, 0, __builtin_amdgcn_readlane(entries, 0), ok0);
    const long g1 = group_of(n, 1, __builtin_amdgcn_readlane(entries, 32), ok1);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int j = i * NT + 64 * wave;
      if (L % NT == 0 || j < L)
        kv[i] = *reinterpret_cast<const uint4v *>(a.kv.codes + (j / (2 * D) ? g1 : g0) * (32 * D) +
                                                  16 * (j % (2 * D)) + 16 * lane);
    }
    there = hh ? ok1 : ok0;
    sc = *reinterpret_cast<const float2v *>(a.kv.scales + 2 * (hh ? g1 : g0));
  };
  auto put_tile = [&](int n, const uint4v (&kv)[NL], float2v sc, bool there) {
    uint8_t *buf = s_kv[n & 3];
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (L % NT == 0 || i * NT + 64 * wave < L) {
        *reinterpret_cast<half8 *>(buf + put0[i]) = codes_f16(kv[i][0], kv[i][1]);
        *reinterpret_cast<half8 *>(buf + put1[i]) = codes_f16(kv[i][2], kv[i][3]);
      }
    // (a group without a page: a value scale of 0, which no group has; every wave writes the same)
    if (i32 == 0) s_sc[n & 3][hh] = there ? sc : float2v{1.0f, 0.0f};
  };
  auto load = [&](int n) {
    fetch_tile(n, ent, raw, raw_sc, raw_there);
    ent = entry(n + 1);
  };
  auto store = [&](int n) { put_tile(n, raw, raw_sc, raw_there); };

  // the first three tiles and the query row, all on their way at once
  half8 qh[TT][2], ql[TT][2];
  int sh;
  {
    const int e0 = entry(0), e1 = entry(1), e2 = entry(2);
    uint4v raw0[NL], raw1[NL];
    float2v sc0, sc1;
    bool there0, there1;
    ent = entry(3);
    fetch_tile(0, e0, raw0, sc0, there0);
    fetch_tile(1, e1, raw1, sc1, there1);
    fetch_tile(2, e2, raw, raw_sc, raw_there);
    const float *row = a.q + (sp.q0 + tq) * a.ldq + (long)head * D;
    const QRope rope = q_rope(a.kv, sp.q0 + tq, sp.p0 + tq);
    float x[TT][16], amax = 0.0f;
    load_q<TT>(row, rope, hh, 2, x);
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(x[t][e]));
    sh = row_shift(max_xor32(amax));
    if (rope.bad) x[0][0] = __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) split_f16(&x[t][8 * u], sh, qh[t][u], ql[t][u]);
    put_tile(0, raw0, sc0, there0);
    put_tile(1, raw1, sc1, there1);
  }
  if (!any) {   // (a wave without rows keeps up the others' tiles and barriers)
    __syncthreads();
    for (int n = 0; n < tiles; ++n) {
      __syncthreads();
      store(n + 2);
      load(n + 3);
    }
    if constexpr (NW == 8) __syncthreads();
    return;
  }

  // A step: tile n's softmax and second product, and with `more` tile n + 1's scores. The matrix instructions
  // of one operand fragment (F of each product, read AHEAD before use) and a share of the vector instructions
  // make a block; the compiler is kept to the order of blocks. (Tiles past the last are loaded as group 0, or what
  // follows it in the table, and never used.)
  //
  // Of 8 waves two share a SIMD. The upper 4 run half a step later, with the step's barrier between its two products
  // where the lower 4 have it before both: one wave's scores stand beside the other's second product and the rest.
  // Between barriers n and n + 1 the lower waves read tiles n + 1 and n, the upper ones n - 1 and n + 1, and both write
  // n + 2: the four of the ring.
  constexpr int F = 2 * TT, AHEAD = 2;
  const int k_at = (hh * 2 * 32 + i32) * 16, v_at = KB + (hh * D + i32) * 16;
  float16v sa, sb;
  float c = 0.0f, lv = 0.0f, rv = 0.0f;   // of the tile whose scores are at hand: factor, log2 and 1 / value scale
  auto step = [&](int n, float16v &s, float16v &s_n, auto has, auto more, auto late) {
    if constexpr (!late.value || !has.value) __syncthreads();
    half8 f[2 * F];   // keys of tile n + 1, values of tile n
    auto fetch = [&](int i) {
      if (i < F)
        f[i] = *reinterpret_cast<const half8 *>(s_kv[(n + 1) & 3] + k_at + (4 * (i >> 1) + (i & 1)) * 32 * 16);
      else
        f[i] = *reinterpret_cast<const half8 *>(s_kv[n & 3] + v_at + (2 * ((i - F) / DT) * D + 32 * ((i - F) % DT)) * 16);
    };
    constexpr int first = more.value ? 0 : F, stop = has.value ? 2 * F : F;
    float2v scale = {1.0f, 0.0f};
    if constexpr (more.value) {
      scale = s_sc[(n + 1) & 3][hh];
#pragma unroll
      for (int e = 0; e < 16; ++e) s_n[e] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(first + i);
    const float shift = (M == kNegInf ? 0.0f : lv - M) + kTop;
    Frag ph[2], pl[2];
    float sum = 0.0f, mx = kNegInf, c_n = 0.0f, lv_n = 0.0f, rv_n = 0.0f;
    bool masked = false;
    if constexpr (!more.value)
#pragma unroll
      for (int p = 0; p < 8; ++p) softmax_pair(s, 2 * p, c, shift, sum, ph, pl);
#pragma unroll
    for (int i = first; i < stop; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (late.value && has.value && i == F) __syncthreads();
      if (i + AHEAD < stop) fetch(i + AHEAD);
      if (i < F) {
        s_n = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i], qh[i >> 1][i & 1], s_n, 0, 0, 0);
        s_n = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i], ql[i >> 1][i & 1], s_n, 0, 0, 0);
      } else {
        const int u = (i - F) / DT, d = (i - F) % DT;
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i], ph[u].h, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i], pl[u].h, o[d], 0, 0, 0);
      }
      if constexpr (has.value && more.value)
#pragma unroll
        for (int p = 0; p < 8; ++p)   // pairs of keys: the first half before the second product starts
          if (i == (p < 4 ? p : 2 * p - 4) * F / 8) softmax_pair(s, 2 * p, c, shift, sum, ph, pl);
      if constexpr (more.value) {
        if (i == F / 2 + 1) {
          float sk = scale[0], sv = scale[1];
          asm volatile("" : "+v"(sk), "+v"(sv));
          masked = (base + 32 * (n + 1) < all_lo) | (base + 32 * (n + 2) > all_hi) | (__ballot(sv == 0.0f) != 0);
          c_n = ldexpf(sk * a.scale2, -sh);   // (as in the 16-row form)
          lv_n = __builtin_amdgcn_logf(sv);
          rv_n = __builtin_amdgcn_rcpf(sv);
          c_n = c_n == 0.0f ? 1e-37f : c_n;   // (a masked score, -inf, stays that)
          asm volatile("" : "+v"(c_n), "+v"(lv_n), "+v"(rv_n));
        }
        if (has.value && i == (late.value ? F : F - 1)) store(n + (late.value ? 3 : 2));
        if (has.value && i == (late.value ? F + 1 : F)) load(n + (late.value ? 4 : 3));
        if (i >= F + F / 2) {
          constexpr int each = 32 / F;
#pragma unroll
          for (int j = each * (i - F - F / 2); j < each * (i - F - F / 2 + 1); ++j) mx = fmaxf(mx, s_n[j]);
          asm volatile("" : "+v"(mx));
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (has.value) l = fmaf(sum * kLow, rv, l);
    if constexpr (more.value) {
      if constexpr (!has.value)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s_n[j]);
      c = c_n;
      lv = lv_n;
      rv = rv_n;
      if (masked) {
        const bool there = scale[1] != 0.0f;
        const int k0 = base + 32 * (n + 1) + 16 * hh, b = see_lo - k0, e = see_hi - k0;
        const uint32_t from = b <= 0 ? 0xffffu : b >= 16 ? 0u : 0xffffu << b;
        const uint32_t to = e <= 0 ? 0u : e >= 16 ? 0xffffu : (1u << e) - 1u;
        const uint32_t on = there ? from & to & 0xffffu : 0u;
        if (on == 0) {   // (a group of which this row sees nothing may hold any scale)
          c = 1.0f;
          lv = rv = 0.0f;
        }
        mx = kNegInf;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          s_n[j] = (on >> j) & 1u ? s_n[j] : kNegInf;
          mx = fmaxf(mx, s_n[j]);
        }
      }
      const float em = max_xor32(fmaf(mx, c, lv));
      if (__ballot(em > M + kSlack)) {
        const float m = em > M + kSlack ? em : M;
        const float2 by = two_factors(M == kNegInf ? kNegInf : M - m);
        const float x = by.x * by.y;
        l = l * by.y * by.x;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= x;
        M = m;
      }
    }
  };
  constexpr std::true_type yes;
  constexpr std::false_type no;
  auto run = [&](auto late) {
    int n = 0;
    step(-1, sb, sa, no, yes, late);
    if constexpr (late.value) {
      __syncthreads();
      store(2);
      load(3);
    }
    for (; n + 2 < tiles; n += 2) {
      step(n, sa, sb, yes, yes, late);
      step(n + 1, sb, sa, yes, yes, late);
    }
    if (n + 1 < tiles) {
      step(n, sa, sb, yes, yes, late);
      step(n + 1, sb, sa, yes, no, late);
    } else if (n < tiles) {
      step(n, sa, sb, yes, no, late);
    }
    if constexpr (NW == 8 && !late.value) __syncthreads();
  };
  if (NW == 8 && wave >= 4) run(yes);
  else run(no);

  if (w0 + i32 > last) return;
  l = kq4_xor_add<32>(l);
  const long row = (long)(sp.q0 + tq) * a.heads + head, n_rows = (long)a.kv.n_tok * a.heads;
  float *dst = used == 1 ? a.out + row * D : part_o(a.part32, n_rows, row, split, D);
  const float f = used > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
  const float low = used > 1 ? 1.0f : kLow;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int j = 0; j < 16; j += 4)
      *reinterpret_cast<float4 *>(dst + 32 * d + 2 * j + 4 * hh) =
          make_float4(o[d][j] * low * f, o[d][j + 1] * low * f, o[d][j + 2] * low * f, o[d][j + 3] * low * f);
  if (used > 1 && hh == 0) *part_ml(a.part32, a.plan.ns32, n_rows, row, split, D) = make_float2(M, l);
}

template <int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_rows16_kernel(AttnArgs a) {
  extern __shared__ __align__(16) uint8_t dyn_lds[];
  attn_rows16<D, NW>(a, blockIdx.x, blockIdx.y, dyn_lds);
}
template <int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_rows32_kernel(AttnArgs a) {
  extern __shared__ __align__(16) uint8_t dyn_lds[];
  attn_rows32<D, NW>(a, blockIdx.x, gridDim.x, blockIdx.y, dyn_lds);
}
// Both in one launch, for batches of short and long runs of tokens: the first blocks16 * ns16 workgroups are
// attn_rows16's, each kind returning for the other's sequences. 7 sequences of 1 to 190 tokens in a window of 1024 of up
// to 2901 keys, 12 heads, 4 kv heads of 64: 21.7 us and 4.7 us for the join, all of it the start and the tiles of the
// longest workgroup (8.8 MB and 2.3 GFLOP would take 2 us).
template <int D>
__global__ __launch_bounds__(256, 2) void attn_mixed_kernel(AttnArgs a, int blocks16, int blocks32) {
  extern __shared__ __align__(16) uint8_t dyn_lds[];
  const int b = blockIdx.x, n16 = blocks16 * a.plan.ns16;
  if (b < n16)
    attn_rows16<D, 4>(a, b % blocks16, b / blocks16, dyn_lds);
  else
    attn_rows32<D, 4>(a, (b - n16) % blocks32, blocks32, (b - n16) / blocks32, dyn_lds);
}

// A row that a thread joins: where its partial sums and its output stand, and how many ranges it has (0: none to join).
struct JoinRow {
  float *part;
  long rows, row, out;
  int n, used;
};

// Row `slot` of the 16-row form's (fewer than 2^18 and a workgroup's); every lane takes part, slots may differ.
KQ4_DEV JoinRow join_row16(const AttnArgs &a, int slot, int lane) {
  const int share = a.plan.deal16 == kShares ? share_turns(a, lane) : 0;
  JoinRow j{a.part16, slots_of(a), slot, 0, a.plan.ns16, 0};
  const int sh = slot / a.plan.cap16, r = slot - sh * a.plan.cap16;
  const int seq = sh / a.kv.kv_heads, h = sh - seq * a.kv.kv_heads;
  if (seq >= a.kv.n_seq) return j;
  const KQ4KvSpan sp = kq4_kv_span(a.kv.q_start[seq], a.kv.q_start[seq + 1], a.kv.kv_len[seq], a.kv.n_tok,
                                   a.kv.table_pages << (a.log_pg + 4));
  const int rows = sp.nq * a.group;
  if (r >= rows || rows > a.plan.cap16 || rows > a.plan.max16) return j;
  int base, end;
  const int r0 = r - r % 16, last = r0 + 15 < rows ? r0 + 15 : rows - 1;
  j.used = kq4_kv_ranges(sp, r0 / a.group, last / a.group, a.window, a.plan.chunk16, a.plan.ns16, &base, &end);
  if (a.plan.deal16 >= kHalves) dealt_part(a, base, end, share, &j.used);
  const int t = r / a.group;
  j.out = (long)(sp.q0 + t) * a.heads + h * a.group + (r - t * a.group);
  return j;
}

// Token tok's row of a head in the 32-row form; tok is the same for the wave, whose lanes all take part.
KQ4_DEV JoinRow join_row32(const AttnArgs &a, int tok, int head, int lane) {
  const long row = (long)tok * a.heads + head;
  JoinRow j{a.part32, (long)a.kv.n_tok * a.heads, row, row, a.plan.ns32, 0};
  for (int b = 0; b < a.kv.n_seq; b += 64) {
    const int i = b + lane;
    KQ4KvSpan t{0, 0, 0, 0};
    if (i < a.kv.n_seq)
      t = kq4_kv_span(a.kv.q_start[i], a.kv.q_start[i + 1], a.kv.kv_len[i], a.kv.n_tok,
                      a.kv.table_pages << (a.log_pg + 4));
    const unsigned long long at = __ballot(tok >= t.q0 && tok < t.q0 + t.nq);
    if (at) {
      const int l = __ffsll((long long)at) - 1;
      const KQ4KvSpan sp{__builtin_amdgcn_readlane(t.q0, l), __builtin_amdgcn_readlane(t.nq, l),
                         __builtin_amdgcn_readlane(t.p0, l), __builtin_amdgcn_readlane(t.len, l)};
      const int rows = sp.nq * a.group;
      if (rows <= a.plan.max16 || head >= a.heads) return j;
      const int r = (tok - sp.q0) * a.group + head % a.group, r0 = r - r % a.plan.tile32;
      const int last = r0 + a.plan.tile32 - 1 < rows ? r0 + a.plan.tile32 - 1 : rows - 1;
      int base, end;
      j.used = kq4_kv_ranges(sp, r0 / a.group, last / a.group, a.window, a.plan.chunk32, a.plan.ns32, &base, &end);
      return j;
    }
  }
  return j;
}

// Joins the splits of rows, few of them: a workgroup takes up to 1024 floats, 4 a thread, of neighbouring rows: blocks16
// workgroups those of the 16-row form, the others `parts` each of a token of the 32-row form. Of a row's 16 or 32 lanes,
// lane s holds split s's factor. Bound by latency (lengths, factors, sums: three dependent loads): 8400 rows of 64, 4
// splits 4.7 us; a wave a row, the factors one after the other, took 7.4.
template <int D>
__global__ __launch_bounds__(256) void attn_join_few_kernel(AttnArgs a, int blocks16, int parts) {
  static_assert(D / 4 >= kJoinFew, "a row's lanes hold a factor each");
  const int lane = threadIdx.x & 63, b = blockIdx.x - blocks16;
  JoinRow j;
  if (b < 0) {
    j = join_row16(a, (int)blockIdx.x * (1024 / D) + 4 * (int)threadIdx.x / D, lane);
  } else {
    const int tok = b / parts;
    j = join_row32(a, tok, (1024 * (b - tok * parts) + 4 * (int)threadIdx.x) / D, lane);
  }
  const int used = j.used, d = 4 * (int)threadIdx.x % D;
  if (used <= 1) return;   // (no row, or written by its only split)
  const int s0 = lane & (kJoinFew - 1);
  const float2 ml = s0 < used ? *part_ml(j.part, j.n, j.rows, j.row, s0, D) : make_float2(kNegInf, 0.0f);
  float m = ml.x;
#pragma unroll
  for (int x = kJoinFew / 2; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  const float2 by = split_factors(ml, m);
  const float f = by.x * by.y;
  float sl = ml.y * by.y * by.x;
#pragma unroll
  for (int x = kJoinFew / 2; x; x >>= 1) sl += __shfl_xor(sl, x);
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  const float *p = part_o(j.part, j.rows, j.row, 0, D) + d;
#pragma unroll 4
  for (int s = 0; s < used; ++s) {
    const float fs = __shfl(f, (lane & -kJoinFew) + s);
    acc += *reinterpret_cast<const float4v *>(p + s * j.rows * D) * fs;
  }
  *reinterpret_cast<float4v *>(a.out + j.out * D + d) = (acc * kLow) * (sl == 0.0f ? 0.0f : 1.0f / sl);
}

// Joins the splits of a row, many of them, 32 dimensions a workgroup (blocks16 of the 16-row form's rows, then the
// 32-row form's): the factors of all splits into LDS, then 8 threads a dimension take splits in turn (32 rows of 128, 64
// splits 4.5 us, latency).
template <int D>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int blocks16) {
  __shared__ float s_f[KQ4_ATTN_MAX_SPLITS];
  __shared__ float s_acc[8][32], s_m[4], s_l[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool few_rows = (int)blockIdx.x < blocks16;
  const int b = few_rows ? blockIdx.x : blockIdx.x - blocks16;
  const long row = b / (D / 32);
  const int d = 32 * (b % (D / 32)) + (tid & 31);
  JoinRow j;
  if (few_rows) {
    j = join_row16(a, (int)row, lane);
  } else {
    const int tok = (int)(row / a.heads);
    j = join_row32(a, tok, (int)(row - (long)tok * a.heads), lane);
  }
  const int used = j.used;
  if (used <= 1) return;
  const float2 *ml0 = part_ml(j.part, j.n, j.rows, j.row, 0, D);

  float m = kNegInf;
  for (int s = tid; s < used; s += 256) m = fmaxf(m, ml0[s * j.rows].x);
#pragma unroll
  for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  if (lane == 0) s_m[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float sl = 0.0f;
  for (int s = tid; s < used; s += 256) {
    const float2 ml = ml0[s * j.rows];
    const float2 f = split_factors(ml, m);
    s_f[s] = f.x * f.y;
    sl = fmaf(ml.y * f.y, f.x, sl);
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) sl += __shfl_xor(sl, x);
  if (lane == 0) s_l[wave] = sl;
  __syncthreads();
  float acc = 0.0f;
  const float *p = part_o(j.part, j.rows, j.row, 0, D) + d;
#pragma unroll 8
  for (int s = tid >> 5; s < used; s += 8) acc = fmaf(p[s * j.rows * D], s_f[s], acc);
  s_acc[tid >> 5][tid & 31] = acc;
  __syncthreads();
  if (tid < 32) {
#pragma unroll
    for (int w = 1; w < 8; ++w) acc += s_acc[w][tid];
    sl = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    a.out[j.out * D + d] = sl == 0.0f ? 0.0f : acc * kLow / sl;
  }
}

// Workgroups of a plan's launches: of each form (times its ranges), and of the joins.
struct Grids {
  long blocks16, blocks32, few16, few32, many16, many32;
};
Grids grids(const KQ4AttnPlan &p, long n_tok, long n_seq, long heads, long kv_heads, long head_dim) {
  const auto few = [](int ns) { return ns > 1 && ns <= kJoinFew; };
  const long floats16 = n_seq * kv_heads * p.cap16 * head_dim, parts = (heads * head_dim + 1023) / 1024;
  return Grids{p.max16 ? (p.deal16 == kShares ? kq4_attn_shares((int)kv_heads, (int)n_seq) + n_seq : n_seq) * kv_heads : 0,
               p.tile32 ? (n_tok * (heads / kv_heads) / p.tile32 + n_seq) * kv_heads : 0,
               few(p.ns16) ? (floats16 + 1023) / 1024 : 0,
               few(p.ns32) ? n_tok * parts : 0,
               p.ns16 > kJoinFew ? floats16 / 32 : 0,
               p.ns32 > kJoinFew ? n_tok * heads * (head_dim / 32) : 0};
}

template <int D>
int launch(const AttnArgs &a, hipStream_t s) {
  const KQ4AttnPlan &p = a.plan;
  const Grids g = grids(p, a.kv.n_tok, a.kv.n_seq, a.heads, a.kv.kv_heads, D);
  const int blocks16 = (int)g.blocks16, blocks32 = (int)g.blocks32;
  const int ns16 = p.deal16 == kShares ? 1 : p.ns16;   // (a range is an item there)
  static std::atomic<unsigned long long> lds8{0}, lds4{0}, ldsm{0};
  constexpr int lds = kLds32<D>;
  hipError_t e = hipSuccess;
  if (p.tile32 == 128 && p.max16) {
    const void *fn = reinterpret_cast<const void *>(&attn_mixed_kernel<D>);
    if ((e = kq4_lds_limit_once(fn, lds, ldsm)) != hipSuccess) return (int)e;
    attn_mixed_kernel<D><<<blocks16 * p.ns16 + blocks32 * p.ns32, 256, lds, s>>>(a, blocks16, blocks32);
  } else {
    if (p.tile32 == 128) {
      const void *fn = reinterpret_cast<const void *>(&attn_rows32_kernel<D, 4>);
      if ((e = kq4_lds_limit_once(fn, lds, lds4)) != hipSuccess) return (int)e;
      attn_rows32_kernel<D, 4><<<dim3(blocks32, p.ns32), 256, lds, s>>>(a);
    } else if (p.tile32) {
      const void *fn = reinterpret_cast<const void *>(&attn_rows32_kernel<D, 8>);
      if ((e = kq4_lds_limit_once(fn, lds, lds8)) != hipSuccess) return (int)e;
      attn_rows32_kernel<D, 8><<<dim3(blocks32, p.ns32), 512, lds, s>>>(a);
    }
    if ((e = hipGetLastError()) != hipSuccess) return (int)e;
    if (p.max16 && p.waves16 == 8) {
      static std::atomic<unsigned long long> lds16{0};
      const void *fn = reinterpret_cast<const void *>(&attn_rows16_kernel<D, 8>);
      if ((e = kq4_lds_limit_once(fn, kLds16<D, 8>, lds16)) != hipSuccess) return (int)e;
      attn_rows16_kernel<D, 8><<<dim3(blocks16, ns16), 512, kLds16<D, 8>, s>>>(a);
    } else if (p.max16) {
      attn_rows16_kernel<D, 4><<<dim3(blocks16, ns16), 256, kLds16<D, 4>, s>>>(a);
    }
  }
  if ((e = hipGetLastError()) != hipSuccess) return (int)e;
  if (g.few16 + g.few32) {
    attn_join_few_kernel<D><<<(unsigned)(g.few16 + g.few32), 256, 0, s>>>(a, (int)g.few16,
                                                                          (int)(((long)a.heads * D + 1023) / 1024));
    if ((e = hipGetLastError()) != hipSuccess) return (int)e;
  }
  if (g.many16 + g.many32) attn_join_kernel<D><<<(unsigned)(g.many16 + g.many32), 256, 0, s>>>(a, (int)g.many16);
  return (int)hipGetLastError();
}

// Splits of `keys` keys so that `base` workgroups become about `want`, each of at least min_chunk keys and at most
// max_chunk (a split's workgroup walks its keys alone, however long other sequences are); none that saves the longest
// workgroup fewer than `save` steps of `step` keys, and never more than `top`.
void split_keys(long keys, long base, int want, int step, int save, int min_chunk, int max_chunk, int force, long top,
                int *chunk, int *ns) {
  long n = want / (base < 1 ? 1 : base);
  const long most = (keys + min_chunk - 1) / min_chunk, least = (keys + max_chunk - 1) / max_chunk;
  if (n > most) n = most;
  const long steps = (keys + step - 1) / step;
  if (n > 1 && steps - (steps + n - 1) / n < save) n = 1;
  if (n < least) n = least;
  if (force > 0) n = force;
  if (n > steps) n = steps;
  if (n > top) n = top;
  if (n > KQ4_ATTN_MAX_SPLITS) n = KQ4_ATTN_MAX_SPLITS;
  if (n < 1) n = 1;
  *chunk = (int)(((keys + n - 1) / n + step - 1) / step * step);
  *ns = (int)((keys + *chunk - 1) / *chunk);
}

// Keys of a tile's queries, at most: the window's reach where that is less.
long most_keys(int max_q, int max_kv, int window) {
  const long keys = max_kv < 1 ? 1 : max_kv > 1 << 30 ? 1 << 30 : max_kv, reach = (long)window + max_q + 64;
  return window > 0 && reach < keys ? reach : keys;
}

}  // namespace

KQ4AttnPlan kq4_attn_plan(int n_tok, int n_seq, int heads, int kv_heads, int max_q, int max_kv, int window,
                          int force_tile, int force_split) {
  const int group = heads / kv_heads;
  const long rows = (long)max_q * group, keys = most_keys(max_q, max_kv, window);
  KQ4AttnPlan p{0, 0, 0, 256, 0, 0, 64, 0, kPlain};
  // 16 rows a tile up to 16 rows of a sequence and kv head (16 sequences of 4 tokens, 4 heads a kv head, 2000 keys:
  // 20.9 us, 39.4 with 128 rows a workgroup; of 8 tokens, 32 rows, 35.7 and 42.6, but one of 16 tokens over 4000 keys
  // 32.8 and 22.8). 256 where its workgroups fill the CUs (a prompt of 4096 tokens 251 us, 277 with 128; 4 of 500 tokens
  // 36.6 and 38.6; one of 2000, whose longest workgroups end late, 95.7 and 85.8), else 128 (the mixed kernel's batch
  // 26.3 us, 30.1 with 256; 500 tokens 26.5 and 32.6).
  p.tile32 = force_tile == 16                                           ? 0
             : force_tile == 128 || force_tile == 256                   ? force_tile
             : rows <= 16                                               ? 0
             : ((long)n_tok * group / 256 + n_seq) * kv_heads >= kCus   ? 256
                                                                        : 128;
  const bool mixed = p.tile32 && force_tile == 0 && n_seq > 1 && (long)n_tok != (long)n_seq * max_q;
  p.max16 = !p.tile32 ? INT_MAX : mixed ? 16 : 0;
  if (p.max16) {
    // 4 waves a workgroup, two of which fit a CU, so that one's start stands beside the other's loads (64 sequences of
    // 1000 keys, 8 kv heads: 25.1 us, 30.9 with 8 waves; 64 of up to 4000 64.8 and 71.0). 8 where there is at most one
    // a CU, by splits or not, and each of its waves has two turns or more (one of 131072 keys, 4 kv heads: 30.0 us,
    // 32.4 with 4 waves; 8 of 8192, 8 kv heads: 29.5 and 32.1; but one of 16384 16.3 and 15.2).
    const long base = (long)n_seq * kv_heads;
    // Room for partial sums: of as many rows as the bounds say a sequence of this form has; longer ones, where a bound
    // is wrong, are not split. (A prompt among decode steps has none here, however many keys they have: one step over
    // 131072 keys beside a chunk of 2048 tokens takes 17 MB.)
    const long room = !mixed ? rows < 1 ? group : rows : group <= 16 ? 16 / group * group : 16;
    p.cap16 = (int)(room < kPartRows ? room : kPartRows);
    const long top = kPartRows / (base * p.cap16);
    const bool full = base >= kCus - kCus / 8;   // the CUs, without splits
    p.waves16 = !mixed && !full && keys / 64 * base > 16 * kCus ? 8 : 4;
    const int turn = 64 * p.waves16;
    // A join costs as much as two turns: 16 sequences, 8 kv heads, 600 / 1000 / 8192 keys in one range 11.2 / 13.4 /
    // 65.5 us, in two 13.4 / 14.6 / 49.2. (At most 1024 keys where the other form's workgroups run beside: 8 sequences
    // of up to 600 tokens and 8000 keys, 16 heads, 355 us, 389 at 512 and at 4096; with 32 heads 533, 535 and 533.)
    split_keys(keys, base, kCus, turn, 3, turn, mixed ? 1024 : 8192, force_split, top, &p.chunk16, &p.ns16);
    // Sequences dealt by length, where there are about as many workgroups as CUs or more and each is long. A CU draws
    // about 30 GB/s whatever is on it, so the time is that of the CU with the most keys: 32 sequences, 8 kv heads, of
    // 1621 to 8192 keys 69.0 -> 59.5 us in halves (the join among it; of 8192 each 85.5 -> 90.9), 28 of up to 8192 66.9
    // -> 59.0 (equal ones 77.6 -> 83.9; but 24 65.0 and 62.0, 73.1 and 79.4: whole, with 8 waves); whole ones in order:
    // 64 of up to 4100 66.8 -> 54.4 (of 4100 each 86.6 -> 89.5), 48 of up to 5000 74.1 -> 55.2, 100 of up to 4500 of 16
    // heads 115 -> 97.
    // Fewer, where the bound makes ranges of 8 turns or more: by shares of all keys that the batch has, up to 4 times
    // an even batch's ranges of a sequence. Finding them costs 2 us (8 sequences of 2000 keys bounded by 32768 21.7 ->
    // 23.8), ranges of the bound far more where it is loose or lengths differ: 8 of up to 8000 bounded by 65536 59.5 ->
    // 30.7 us, one of 16384 bounded by 131072 35.7 -> 19.2. Between half and 7/8 of the CUs neither rule applies and each
    // sequence is one range: 17 of up to 8192 keys take 62 us, 46.7 in 4 ranges each; 17 equal ones 67.0 and 69.1.
    if (!mixed && force_split <= 0 && base <= kCus / 2 && p.ns16 > 1 && p.chunk16 >= 8 * turn) {
      p.deal16 = kShares;
      const long most = 4 * (kCus / base), have = (keys + turn - 1) / turn, places = kCus / kv_heads;
      p.ns16 = (int)(most < have ? most : have);
      if (p.ns16 > places) p.ns16 = (int)places;
      if (p.ns16 > top) p.ns16 = (int)top;
    } else if (!mixed && force_split <= 0 && full && n_seq <= 64 * p.waves16 && keys >= 16 * turn) {
      if (base > kCus && p.ns16 == 1) p.deal16 = kOrder;
      if (base <= kCus && p.ns16 <= 2 && top > 1) {
        p.deal16 = kHalves;
        p.ns16 = 2;
      }
    }
  }
  if (p.tile32) {
    // A split more saves the longest workgroup tiles of keys (about 0.9 us each) and costs every row a partial sum
    // written and read: keys / n + n rows / kRowKeys is least at n^2 = kRowKeys keys / rows. (kRowKeys 40 / 80 / 140:
    // 64 tokens x 32 heads over 2000 keys 27.9 / 25.8 / 26.5 us, 3 x 200 x 8 over 400 24.7 / 23.6 / 23.5, 4 x 100 x 16
    // over 900 32.9 / 29.4 / 32.0.)
    const int best = (int)(sqrt((double)kRowKeys * keys / ((double)n_tok * heads)) + 0.5);
    const long least = best < 2 ? keys : (keys + best - 1) / best;
    split_keys(keys, ((long)n_tok * group + p.tile32 - 1) / p.tile32 * kv_heads, p.tile32 == 128 ? 2 * kCus : kCus,
               64, 0, least > kMinChunk ? (int)least : kMinChunk, INT_MAX, force_split, LONG_MAX, &p.chunk32, &p.ns32);
  }
  return p;
}

namespace {

size_t part_bytes(long rows, int head_dim) {   // (a multiple of 256)
  return ((size_t)rows * (head_dim * sizeof(float) + sizeof(float2)) + 255) & ~(size_t)255;
}

}  // namespace

size_t kq4_attn_part_bytes(const KQ4AttnPlan &p, int n_tok, int n_seq, int heads, int kv_heads, int head_dim,
                           size_t *bytes16) {
  *bytes16 = p.ns16 > 1 ? part_bytes((long)p.ns16 * n_seq * kv_heads * p.cap16, head_dim) : 0;
  return *bytes16 + (p.ns32 > 1 ? part_bytes((long)p.ns32 * n_tok * heads, head_dim) : 0);
}

// No batch of at most these numbers has more: the 16-row form makes of `base` workgroups at most kCus by its splits,
// 4 kCus by shares, or as many as its longest range allows, of at least 4 turns of 256 keys; the 32-row form 2 kCus of
// 128 rows or kCus of 256.
size_t kq4_attn_most_part_bytes(int n_tok, int n_seq, int heads, int kv_heads, int head_dim, int max_q, int max_kv,
                                int window, int force_tile, int force_split) {
  const long group = heads / kv_heads, rows = max_q * group, keys = most_keys(max_q, max_kv, window);
  const long base = (long)n_seq * kv_heads, turns = (keys + 255) / 256;
  long rows16 = 0, rows32 = 0;
  if (force_tile != 128 && force_tile != 256) {
    const long tile = group > 16 ? group : 16, cap = rows < 1 ? group : force_tile == 16 || rows < tile ? rows : tile;
    const long longest = rows > 16 ? 1024 : 8192, least = (keys + longest - 1) / longest;
    long ranges = base * least > 4 * kCus ? base * least : 4 * kCus;
    if (base * turns < ranges) ranges = base * turns;
    if (force_split > 0) ranges = base * (force_split < turns ? force_split : turns);
    else if (turns < 4) ranges = 0;
    rows16 = ranges * cap < kPartRows ? ranges * cap : kPartRows;
  }
  if (force_tile == 128 || force_tile == 256 || (force_tile != 16 && rows > 16)) {
    const long all = (long)n_tok * heads, steps = (keys + 63) / 64;
    long n = force_split < steps ? force_split : steps;
    if (n > KQ4_ATTN_MAX_SPLITS) n = KQ4_ATTN_MAX_SPLITS;
    rows32 = force_split > 0 ? all * n : keys > kMinChunk ? all * ((keys + kMinChunk - 1) / kMinChunk) : 0;
    if (force_split <= 0 && rows32 > kCus * 256) rows32 = kCus * 256;
  }
  return part_bytes(rows16, head_dim) + part_bytes(rows32, head_dim);
}

bool kq4_attn_fits(const KQ4AttnPlan &p, int n_tok, int n_seq, int heads, int kv_heads, int head_dim) {
  const Grids g = grids(p, n_tok, n_seq, heads, kv_heads, head_dim);
  const long forms = p.tile32 == 256 || p.waves16 == 8 ? 512 : 256, most = 0xffffffffL;
  return (g.blocks16 * p.ns16 + g.blocks32 * p.ns32) * forms <= most && (g.few16 + g.few32) * 256 <= most &&
         (g.many16 + g.many32) * 256 <= most;
}

int kq4_launch_attn(float *out, const kq4_kv &kv, int log_pg, const float *q, long ldq, int heads, float scale,
                    int window, const KQ4AttnPlan &plan, char *ws, hipStream_t s) {
  size_t at;
  const bool split = kq4_attn_part_bytes(plan, kv.n_tok, kv.n_seq, heads, kv.kv_heads, kv.head_dim, &at) > 0;
  AttnArgs a{kv, q, ldq, out, log_pg, heads, heads / kv.kv_heads, scale * 1.44269504088896340736f, window, plan,
             reinterpret_cast<float *>(ws), reinterpret_cast<float *>(split ? ws + at : ws)};
  return kv.head_dim == 128 ? launch<128>(a, s) : launch<64>(a, s);
}
