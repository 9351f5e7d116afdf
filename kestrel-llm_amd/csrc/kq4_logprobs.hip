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
// reach the n_top-th largest of the threads' own maxima (there are at least n_top of those, and few more in
// most rows), ordered by rank counting. Rows where many elements tie for it are selected exactly instead,
// by bisection of the key and then of the index.
// The order is that of the key: the logit's, ties to the lowest index; -inf is never a candidate.
#include "kq4_common.h"
#include "kq4_internal.h"

namespace {

constexpr int kThreads = 256, kPer = 32, kPiece = kThreads * kPer, kCand = 512;
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

KQ4_DEV float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
KQ4_DEV float wave_max(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

struct Piece {   // of one row: maximum, z and t relative to it, whether it has a NaN
  float m, z, t;
  uint32_t nan;
};

// Element i of a thread is logit base + at(i).
template <bool V4>
KQ4_DEV int at(int i) {
  return V4 ? (i >> 2) * (4 * kThreads) + 4 * (int)threadIdx.x + (i & 3) : i * kThreads + (int)threadIdx.x;
}

template <bool V4>
__global__ __launch_bounds__(kThreads) void logprobs_piece_kernel(const float *__restrict__ logits, long ld,
                                                                  int vocab, int n_pieces, int n_top, Piece *__restrict__ pieces,
                                                                  unsigned long long *__restrict__ best) {
  __shared__ float s_m[4], s_z[4], s_t[4];
  __shared__ __align__(16) uint32_t s_keys[kThreads];
  __shared__ uint32_t s_nan[4], s_thr;
  __shared__ int s_ones[4], s_count[4];
  __shared__ int s_n;
  __shared__ unsigned long long s_cand[kCand];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / n_pieces, piece = blockIdx.x - row * n_pieces, base = piece * kPiece;
  const float *x = logits + row * ld + base;
  const int n = vocab - base < kPiece ? vocab - base : kPiece;

  float v[kPer];
  if constexpr (V4) {
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const int o = at<V4>(i);
      float4 f = make_float4(kNegInf, kNegInf, kNegInf, kNegInf);
      if (o + 4 <= n) {
        f = *reinterpret_cast<const float4 *>(x + o);
      } else if (o < n) {
        f.x = x[o];
        if (o + 1 < n) f.y = x[o + 1];
        if (o + 2 < n) f.z = x[o + 2];
      }
      v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = at<V4>(i) < n ? x[at<V4>(i)] : kNegInf;
  }

  float mt = kNegInf;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    mt = fmaxf(mt, v[i]);
    nan |= v[i] != v[i];
  }
  const float mw = wave_max(mt);
  const bool nw = __ballot(nan) != 0;
  if (lane == 0) {
    s_m[wave] = mw;
    s_nan[wave] = nw;
  }
  s_keys[tid] = nan ? 0xffffffffu : key_of(mt);
  if (tid == 0) {
    s_thr = 0;
    s_n = 0;
  }
  __syncthreads();
  const float m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));

  // the maximum's elements are counted, the others summed
  float z = 0.0f, t = 0.0f;
  int ones = 0;
  if (m > kNegInf) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float d = fmaxf(v[i] - m, kFar);
      const float e = v[i] == m ? 0.0f : __builtin_amdgcn_exp2f(d * kLog2e);
      ones += v[i] == m;
      z += e;
      t = fmaf(e, d, t);
    }
  }
  z = wave_sum(z);
  t = wave_sum(t);
#pragma unroll
  for (int x2 = 32; x2; x2 >>= 1) ones += __shfl_xor(ones, x2);
  if (lane == 0) {
    s_z[wave] = z;
    s_t[wave] = t;
    s_ones[wave] = ones;
  }
  unsigned long long *out = best + (long)blockIdx.x * n_top;

  if (n_top > 0) {
    // the n_top-th largest of the threads' maxima
    const uint32_t mine = s_keys[tid];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < kThreads; j += 4) {
      const uint4 k = *reinterpret_cast<const uint4 *>(&s_keys[j]);
      above += (k.x > mine || (k.x == mine && j < tid)) + (k.y > mine || (k.y == mine && j + 1 < tid)) +
               (k.z > mine || (k.z == mine && j + 2 < tid)) + (k.w > mine || (k.w == mine && j + 3 < tid));
    }
    if (above == n_top - 1) s_thr = mine > kKeyNegInf ? mine : kKeyNegInf + 1;
    __syncthreads();
    const uint32_t thr = s_thr;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t k = key_of(v[i]);
      const unsigned long long in = __ballot(k >= thr);
      if (in) {
        int first = 0;
        if (lane == 0) first = atomicAdd(&s_n, (int)__popcll(in));
        first = __builtin_amdgcn_readfirstlane(first);
        const int slot = first + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
        if (k >= thr && slot < kCand) s_cand[slot] = ((unsigned long long)k << 32) | (uint32_t)~(base + at<V4>(i));
      }
    }
    __syncthreads();
    int nc = s_n;
    if (nc > kCand) {
      // too many ties: the n_top-th key by bisection, then how far into its equals
      auto count = [&](auto pred) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) c += (int)__popcll(__ballot(pred(i)));
        __syncthreads();
        if (lane == 0) s_count[wave] = c;
        __syncthreads();
        return s_count[0] + s_count[1] + s_count[2] + s_count[3];
      };
      uint32_t lo = thr, hi = 0xffffffffu;   // the largest key that at least n_top elements reach
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        if (count([&](int i) { return key_of(v[i]) >= mid; }) >= n_top) lo = mid;
        else hi = mid - 1;
      }
      const int more = count([&](int i) { return key_of(v[i]) > lo; });
      int a = 0, b = kPiece - 1;             // the smallest end that leaves n_top - more equals
      while (a < b) {
        const int mid = (a + b) / 2;
        if (count([&](int i) { return key_of(v[i]) == lo && at<V4>(i) <= mid; }) >= n_top - more) b = mid;
        else a = mid + 1;
      }
      if (tid == 0) s_n = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t k = key_of(v[i]);
        if (k > lo || (k == lo && at<V4>(i) <= a))
          s_cand[atomicAdd(&s_n, 1)] = ((unsigned long long)k << 32) | (uint32_t)~(base + at<V4>(i));
      }
      __syncthreads();
      nc = s_n;
    }
    for (int c = tid; c < nc; c += kThreads) {
      const unsigned long long mine2 = s_cand[c];
      int rank = 0;
      for (int j = 0; j < nc; ++j) rank += s_cand[j] > mine2;
      if (rank < n_top) out[rank] = mine2;
    }
    for (int j = nc + tid; j < n_top; j += kThreads) out[j] = 0;
  } else {
    __syncthreads();
  }
  if (tid == 0) {
    Piece p;
    p.m = m;
    p.z = 0.0f;
    p.t = 0.0f;
    p.nan = s_nan[0] | s_nan[1] | s_nan[2] | s_nan[3];
    if (m > kNegInf) {
      p.z = ((s_z[0] + s_z[1]) + (s_z[2] + s_z[3])) + (float)(s_ones[0] + s_ones[1] + s_ones[2] + s_ones[3] - 1);
      p.t = (s_t[0] + s_t[1]) + (s_t[2] + s_t[3]);
    }
    pieces[blockIdx.x] = p;
  }
}

// Joins a row's pieces, one wave a row.
__global__ __launch_bounds__(64) void logprobs_join_kernel(const float *__restrict__ logits, long ld, int vocab,
                                                           int n_pieces, int n_top, const int *__restrict__ token,
                                                           const Piece *__restrict__ pieces,
                                                           const unsigned long long *__restrict__ best,
                                                           float *logprob, float *entropy, float *top_logprob,
                                                           int *top_id) {
  extern __shared__ unsigned long long s_list[];
  const int lane = threadIdx.x;
  const long row = blockIdx.x;
  const Piece *p = pieces + row * n_pieces;

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
  if (lane == 0) {
    if (logprob) {
      const int id = token[row];
      float r = bad;
      if (id >= 0 && id < vocab && !nan) r = M > kNegInf ? (logits[row * ld + id] - M) - lz : kNegInf;
      logprob[row] = r;
    }
    if (entropy) entropy[row] = nan ? bad : M > kNegInf ? lz - t / (1.0f + z) : 0.0f;
  }
  if (n_top == 0) return;

  // each of the pieces has ceil(n_top / n_pieces) elements that reach the least of those
  const unsigned long long *l = best + row * n_pieces * n_top;
  const int q = (n_top + n_pieces - 1) / n_pieces;
  unsigned long long thr = ~0ull;
  for (int i = lane; i < n_pieces; i += 64) {
    const unsigned long long e = l[(long)i * n_top + q - 1];
    thr = e < thr ? e : thr;
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) {
    const unsigned long long o = __shfl_xor(thr, x);
    thr = o < thr ? o : thr;
  }
  int nc = 0;
  for (int b = 0; b < n_pieces * n_top; b += 64) {
    const unsigned long long e = b + lane < n_pieces * n_top ? l[b + lane] : 0;
    const bool in = e != 0 && e >= thr;
    const unsigned long long all = __ballot(in);
    if (in) s_list[nc + (int)__popcll(all & ((1ull << lane) - 1))] = e;
    nc += (int)__popcll(all);
  }
  __syncthreads();
  float *out_lp = top_logprob + row * n_top;
  int *out_id = top_id + row * n_top;
  for (int c = lane; c < nc; c += 64) {
    const unsigned long long e = s_list[c];
    int rank = 0;
    for (int j = 0; j < nc; ++j) rank += s_list[j] > e;
    if (rank < n_top) {
      out_lp[rank] = nan ? bad : (key_value((uint32_t)(e >> 32)) - M) - lz;
      out_id[rank] = (int)~(uint32_t)e;
    }
  }
  if (nc < n_top) {   // the lowest ids of those at -inf (n_top <= 32: the first 64 ids hold enough)
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
  if ((uintptr_t)logits % 16 == 0 && ld % 4 == 0)
    logprobs_piece_kernel<true><<<grid, kThreads, 0, s>>>(logits, ld, vocab, np, n_top, pc, best);
  else
    logprobs_piece_kernel<false><<<grid, kThreads, 0, s>>>(logits, ld, vocab, np, n_top, pc, best);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  logprobs_join_kernel<<<(unsigned)n, 64, (size_t)np * n_top * sizeof(unsigned long long), s>>>(
      logits, ld, vocab, np, n_top, token, pc, best, logprob, entropy, top_logprob, top_id);
  return (int)hipGetLastError();
}
