// kq4_logprobs.hip - log probabilities of given tokens, entropy and top alternatives of rows of logits.
//
// With m a row's maximum, z = sum over every element but one that has it of e^(x - m) and
// t = sum of e^(x - m) (x - m):
//   log p_i = x_i - m - log1p(z),   entropy = log1p(z) - t / (1 + z)
// Leaving the maximum's own 1 out of z keeps the digits of a sure row (z far below 1), and both terms of the
// entropy are at least 0, so nothing cancels.
//
// One pass: a workgroup holds 8192 logits of a row in registers (32 a thread), reduces its (m, z, t) and
// picks its n_top best; a second launch joins a row's pieces. Candidates for the best are the elements that
// reach a threshold that at least n_top elements reach: the n_top-th largest of the threads' maxima, to 16 bits, by
// bisection in one wave while the others sum. Few others reach it in most rows (of 8192 normal ones about 21 the
// largest 20 of 256 maxima). They are ordered by rank counting. Rows where too many elements reach it (many equal
// ones), and rows with a NaN, are selected exactly instead, by bisection of the key and then of the index.
// The order is that of the key: the logit's, ties to the lowest index; -inf is never a candidate.
// Bound by memory for many rows: 1000 rows of 128003 (512 MB) 77 us and 5 for the join, 6.2 TB/s (loads that leave the
// caches alone; 93 us in all with ordinary ones). 64 rows of 151936, 20 best: 13.5 and 4.8 us, of which the loads take
// about 8: all workgroups are resident at once, so the sums and the selection (3.5 us) stand behind the loads. One row:
// 5.9 and 4.0 us, latency of two launches. Pieces of 8192: 32 logits a thread keep 8 loads of 16 bytes in flight.
#include "kq4_common.h"
#include "kq4_internal.h"
#include "../../include/kq4.h"

namespace {

constexpr int kThreads = 256, kPer = 32, kPiece = kThreads * kPer, kCand = 128;   // (kCand: a wave's)
constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kFar = -1000.0f;   // e^d is 0 long before; no product of it with a 0 or a sum overflows
constexpr uint32_t kKeyNegInf = 0x007fffffu;   // key of -inf; 0: no element

// Order-preserving key of a logit; -0 as +0, a NaN above everything.
KQ4_DEV uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return x != x ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
KQ4_DEV float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// A wave's sum or maximum in every lane: DPP moves within rows of 16 lanes, then the swaps of rows and halves. (Rotations
// add a row's quads in an order of each lane's own, so a sum of floats is lane 0's for all: results that lanes form with
// it must not depend on which lane does.)
template <int CTRL>
KQ4_DEV uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
constexpr int kQuad1 = 0xB1, kQuad2 = 0x4E, kRow4 = 0x124, kRow8 = 0x128;   // xor 1, xor 2, rotate by 4, by 8
KQ4_DEV float wave_sum(float v) {
  v += __uint_as_float(dpp<kQuad1>(__float_as_uint(v)));
  v += __uint_as_float(dpp<kQuad2>(__float_as_uint(v)));
  v += __uint_as_float(dpp<kRow4>(__float_as_uint(v)));
  v += __uint_as_float(dpp<kRow8>(__float_as_uint(v)));
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(kq4_xor_add<32>(kq4_xor_add<16>(v)))));
}
KQ4_DEV int wave_sum(int n) {
  uint32_t v = (uint32_t)n;
  v += dpp<kQuad1>(v);
  v += dpp<kQuad2>(v);
  v += dpp<kRow4>(v);
  v += dpp<kRow8>(v);
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = r[0] + r[1];
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return (int)(r[0] + r[1]);
}
KQ4_DEV float wave_max(float v) {
  v = kq4_max32(v);
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

struct Piece {   // of one row: maximum, z and t relative to it, whether it has a NaN
  float m, z, t;
  uint32_t nan;
};

// Element i of a thread is logit base + at(i).
KQ4_DEV int at(int i) { return (i >> 2) * (4 * kThreads) + 4 * (int)threadIdx.x + (i & 3); }

typedef float four __attribute__((ext_vector_type(4), aligned(4)));   // 16 bytes at any 4-byte address

__global__ __launch_bounds__(kThreads) void logprobs_piece_kernel(const float *__restrict__ logits, long ld,
                                                                  int vocab, int n_pieces, int n_top,
                                                                  Piece *__restrict__ pieces,
                                                                  unsigned long long *__restrict__ best) {
  __shared__ float s_m[4], s_z[4], s_t[4], s_thr;
  __shared__ int s_ones[4], s_count[4];
  __shared__ int s_n;
  __shared__ __align__(16) uint32_t s_key[kThreads];
  __shared__ __align__(16) unsigned long long s_cand[4][kCand];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x / n_pieces, piece = blockIdx.x - row * n_pieces, base = piece * kPiece;
  const float *x = logits + row * ld + base;
  const int n = vocab - base < kPiece ? vocab - base : kPiece;

  float v[kPer];
  if (n == kPiece) {
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const four f = __builtin_nontemporal_load(reinterpret_cast<const four *>(x + at(i)));
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i + j] = f[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const int o = at(i);
      four f = {kNegInf, kNegInf, kNegInf, kNegInf};
      if (o + 4 <= n) {
        f = *reinterpret_cast<const four *>(x + o);
      } else {
        if (o < n) f[0] = x[o];
        if (o + 1 < n) f[1] = x[o + 1];
        if (o + 2 < n) f[2] = x[o + 2];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i + j] = f[j];
    }
  }

  float mt = v[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) mt = fmaxf(mt, v[i]);
  const float mw = wave_max(mt);
  if (lane == 0) s_m[wave] = mw;
  s_key[tid] = key_of(mt);
  __syncthreads();
  const float m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  if (wave == 0 && n_top > 0) {
    // a value that n_top threads' maxima reach, 16 bits of the largest such key (or the least number, where fewer have
    // anything but -inf: then every such element, up to the limit)
    const uint4 k = *reinterpret_cast<const uint4 *>(&s_key[4 * lane]);
    uint32_t reach = 0;
#pragma unroll
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
      const uint32_t c = reach | bit;
      if ((int)(__popcll(__ballot(k.x >= c)) + __popcll(__ballot(k.y >= c)) + __popcll(__ballot(k.z >= c)) +
                __popcll(__ballot(k.w >= c))) >= n_top)
        reach = c;
    }
    if (lane == 0) s_thr = reach > kKeyNegInf ? key_value(reach) : -__FLT_MAX__;
  }

  // the maximum's elements are counted, the others summed (only a wave that has it looks for them)
  float z = 0.0f, t = 0.0f;
  int ones = 0;
  if (m > kNegInf) {
    if (mw == m) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float d = v[i] - m;
        const float e = d == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(d * kLog2e);
        ones += d == 0.0f;
        z += e;
        t = fmaf(e, fmaxf(d, kFar), t);
      }
      ones = wave_sum(ones);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float d = v[i] - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
        z += e;
        t = fmaf(e, fmaxf(d, kFar), t);
      }
    }
    z = wave_sum(z);   // (a NaN among the logits makes it NaN; the maxima pass over it)
    t = wave_sum(t);
  } else {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) nan |= v[i] != v[i];
    if (__ballot(nan)) z = __uint_as_float(0x7fc00000u);
  }
  if (lane == 0) {
    s_z[wave] = z;
    s_t[wave] = t;
    s_ones[wave] = ones;
  }
  __syncthreads();
  const bool has_nan = !(s_z[0] + s_z[1] + s_z[2] + s_z[3] >= 0.0f);
  if (n_top > 0) {
    unsigned long long *out = best + (long)blockIdx.x * n_top;
    const float thr = s_thr;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool in = v[i] >= thr;
      const unsigned long long all = __ballot(in);
      if (all) {
        const int slot = c + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32),
                                                            __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
        if (in && slot < kCand) s_cand[wave][slot] = ((unsigned long long)key_of(v[i]) << 32) | (uint32_t)~(base + at(i));
        c += (int)__popcll(all);
      }
    }
    if (lane == 0) s_count[wave] = c;
    __syncthreads();
    int n0 = s_count[0], n1 = s_count[1], n2 = s_count[2], n3 = s_count[3];
    if (n0 > kCand || n1 > kCand || n2 > kCand || n3 > kCand || has_nan) {
      // the n_top-th key by bisection, then how far into its equals
      auto count = [&](auto pred) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) c += pred(i);
        c = wave_sum(c);
        __syncthreads();
        if (lane == 0) s_count[wave] = c;
        __syncthreads();
        return s_count[0] + s_count[1] + s_count[2] + s_count[3];
      };
      uint32_t lo = kKeyNegInf + 1, hi = 0xffffffffu;   // the largest key that at least n_top elements reach
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        if (count([&](int i) { return key_of(v[i]) >= mid; }) >= n_top) lo = mid;
        else hi = mid - 1;
      }
      const int more = count([&](int i) { return key_of(v[i]) > lo; });
      int a = 0, b = kPiece - 1;             // the smallest end that leaves n_top - more equals
      while (a < b) {
        const int mid = (a + b) / 2;
        if (count([&](int i) { return key_of(v[i]) == lo && at(i) <= mid; }) >= n_top - more) b = mid;
        else a = mid + 1;
      }
      if (tid == 0) s_n = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) {       // (n_top elements, or fewer where there are no more than that)
        const uint32_t k = key_of(v[i]);
        if (k > lo || (k == lo && at(i) <= a))
          s_cand[0][atomicAdd(&s_n, 1)] = ((unsigned long long)k << 32) | (uint32_t)~(base + at(i));
      }
      __syncthreads();
      n0 = s_n;
      n1 = n2 = n3 = 0;
    }
    const int nc = n0 + n1 + n2 + n3;
    for (int i = tid; i < nc; i += kThreads) {
      int w = 0, j = i;   // entry j of wave w's
      if (j >= n0) { j -= n0; w = 1; }
      if (w == 1 && j >= n1) { j -= n1; w = 2; }
      if (w == 2 && j >= n2) { j -= n2; w = 3; }
      const unsigned long long mine = s_cand[w][j];
      int rank = 0;
      for (int q = 0; q < n0; ++q) rank += s_cand[0][q] > mine;
      for (int q = 0; q < n1; ++q) rank += s_cand[1][q] > mine;
      for (int q = 0; q < n2; ++q) rank += s_cand[2][q] > mine;
      for (int q = 0; q < n3; ++q) rank += s_cand[3][q] > mine;
      if (rank < n_top) out[rank] = mine;
    }
    for (int j = nc + tid; j < n_top; j += kThreads) out[j] = 0;
  }
  if (tid == 0) {
    Piece p{m, 0.0f, 0.0f, has_nan};
    if (m > kNegInf) {
      p.z = ((s_z[0] + s_z[1]) + (s_z[2] + s_z[3])) + (float)(s_ones[0] + s_ones[1] + s_ones[2] + s_ones[3] - 1);
      p.t = (s_t[0] + s_t[1]) + (s_t[2] + s_t[3]);
    }
    pieces[blockIdx.x] = p;
  }
}

// Joins a row's pieces, a workgroup a row (each wave forms the sums for itself).
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(const float *__restrict__ logits, long ld, int vocab,
                                                           int n_pieces, int n_top, const int *__restrict__ token,
                                                           const Piece *__restrict__ pieces,
                                                           const unsigned long long *__restrict__ best,
                                                           float *logprob, float *entropy, float *top_logprob,
                                                           int *top_id) {
  extern __shared__ unsigned long long s_list[];
  __shared__ int s_n;
  __shared__ unsigned long long s_thr;
  const int tid = threadIdx.x, lane = tid & 63;
  const long row = blockIdx.x;
  const Piece *p = pieces + row * n_pieces;
  const int id = logprob ? token[row] : -1;
  const float at_id = id >= 0 && id < vocab ? logits[row * ld + id] : 0.0f;
  // the pieces' lists, each sorted (0: no element), behind the room for those that are kept
  unsigned long long *s_all = s_list + n_pieces * n_top;
  if (tid == 0) {
    s_n = 0;
    s_thr = 0;
  }
  for (int i = tid; i < n_pieces * n_top; i += kThreads) s_all[i] = best[row * n_pieces * n_top + i];

  float M = kNegInf;
  bool nan = false;
  for (int i = lane; i < n_pieces; i += 64) {
    M = fmaxf(M, p[i].m);
    nan |= p[i].nan != 0;
  }
  M = wave_max(M);
  nan = __ballot(nan) != 0 || M == __builtin_inff();
  // each piece's maximum is 1 in its own z + 1; the first piece that has the row's is the one left out
  float z = 0.0f, t = 0.0f;
  bool owned = false;
  for (int b = 0; b < n_pieces; b += 64) {
    const int i = b + lane;
    const Piece q = i < n_pieces ? p[i] : Piece{kNegInf, 0.0f, 0.0f, 0};
    const unsigned long long has = __ballot(q.m == M && i < n_pieces);
    const bool owner = !owned && has && lane == __ffsll((long long)has) - 1;
    owned |= has != 0;
    if (q.m > kNegInf) {
      const float d = fmaxf(q.m - M, kFar), f = __builtin_amdgcn_exp2f(d * kLog2e);
      z += owner ? q.z : (q.z + 1.0f) * f;
      t += owner ? q.t : f * fmaf(q.z + 1.0f, d, q.t);
    }
  }
  z = wave_sum(z);
  t = wave_sum(t);
  const float bad = __uint_as_float(0x7fc00000u), lz = log1pf(z);
  if (tid == 0) {
    if (logprob) {
      float r = bad;
      if (id >= 0 && id < vocab && !nan) r = M > kNegInf ? (at_id - M) - lz : kNegInf;
      logprob[row] = r;
    }
    if (entropy) entropy[row] = nan ? bad : M > kNegInf ? lz - t / (1.0f + z) : 0.0f;
  }
  if (n_top == 0) return;

  // at least n_top elements reach the `lists`-th largest of the lists' q-th elements
  int q = n_top < 4 ? n_top : 4;
  if (q * n_pieces < n_top) q = (n_top + n_pieces - 1) / n_pieces;
  const int lists = (n_top + q - 1) / q;
  __syncthreads();
  if (tid < n_pieces) {
    const unsigned long long e = s_all[tid * n_top + q - 1];
    int above = 0;
    for (int j = 0; j < n_pieces; ++j) above += s_all[j * n_top + q - 1] > e;
    if (e != 0 && above == lists - 1) s_thr = e;
  }
  __syncthreads();
  const unsigned long long thr = s_thr;
  for (int i = tid; i < n_pieces * n_top; i += kThreads) {
    const unsigned long long e = s_all[i];
    if (e != 0 && e >= thr) s_list[atomicAdd(&s_n, 1)] = e;
  }
  __syncthreads();
  const int nc = s_n;
  float *out_lp = top_logprob + row * n_top;
  int *out_id = top_id + row * n_top;
  for (int c = tid; c < nc; c += kThreads) {
    const unsigned long long e = s_list[c];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < nc; ++j) rank += s_list[j] > e;
    if (rank < n_top) {
      out_lp[rank] = nan ? bad : (key_value((uint32_t)(e >> 32)) - M) - lz;
      out_id[rank] = (int)~(uint32_t)e;
    }
  }
  if (nc < n_top && tid < 64) {   // the lowest ids of those at -inf (n_top <= 32: the first 64 ids hold enough)
    bool taken = lane >= vocab;
    for (int j = 0; j < nc; ++j) taken |= (int)~(uint32_t)s_list[j] == lane;
    const unsigned long long open = __ballot(!taken);
    const int rank = nc + (int)__popcll(open & ((1ull << lane) - 1));
    if (!taken && rank < n_top) {
      out_lp[rank] = nan ? bad : kNegInf;
      out_id[rank] = lane;
    }
  }
}

}  // namespace

int kq4_logprobs_pieces(int vocab) { return (vocab + kPiece - 1) / kPiece; }
size_t kq4_logprobs_piece_bytes() { return sizeof(Piece); }

int kq4_launch_logprobs(const float *logits, long ld, int n, int vocab, int n_top, const int *token, float *logprob,
                        float *entropy, float *top_logprob, int *top_id, void *pieces, unsigned long long *best,
                        hipStream_t s) {
  const int np = kq4_logprobs_pieces(vocab);
  Piece *pc = static_cast<Piece *>(pieces);
  const unsigned grid = (unsigned)((long)n * np);
  logprobs_piece_kernel<<<grid, kThreads, 0, s>>>(logits, ld, vocab, np, n_top, pc, best);
  static std::atomic<unsigned long long> limit{0};
  constexpr int most = 2 * (KQ4_LOGPROBS_MAX_VOCAB / kPiece) * KQ4_LOGPROBS_MAX_TOP * (int)sizeof(unsigned long long);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) e = kq4_lds_limit_once(reinterpret_cast<const void *>(&logprobs_join_kernel), most, limit);
  if (e != hipSuccess) return (int)e;
  logprobs_join_kernel<<<(unsigned)n, kThreads, 2 * (size_t)np * n_top * sizeof(unsigned long long), s>>>(
      logits, ld, vocab, np, n_top, token, pc, best, logprob, entropy, top_logprob, top_id);
  return (int)hipGetLastError();
}
