// kq4_mx_rows.hip - products of few tokens with 4-bit microscaled weights.
//   out[t][r] = [res[t][r] +] sum_k x[t][k] w[r][k]                    (G = 1)
//   out[t][r] = silu(sum_k x[t][k] wg[r][k]) * sum_k x[t][k] wu[r][k]  (G = 2)
#include "kq4_internal.h"
#include "kq4_mx_dev.h"

// A wave takes RT row tiles of 16 rows (of each matrix) against 16 * TT tokens and every KS-th piece of 512 columns (a
// dword of scales per lane, a byte for each 128 of them); KS waves of a workgroup share row tiles, and their sums are
// added in LDS in wave order. The weights, read once, go from memory to the registers of
// v_mfma_scale_f32_16x16x128_f8f6f4 as they lie, a tile one 16-byte load per lane.
// The activations come the same way from a quantized matrix (FQ = 0), or the workgroup quantizes the fp32 rows into LDS
// while its first weights are on their way (FQ = 1): one launch instead of two. Loads return in order, so what is needed
// first is asked for first: the activations before the weights. What bounds it: the weights' bytes where they are many (one
// token: 151936 x 2048 27 us, 6.1 TB/s; 2 x 12288 x 4096 gated 11 us, 4.9 TB/s with what starts and ends it), the latency of
// a piece below (4096 x 4096 4.4 us), the operands' way through the L2 caches for more tokens (64 x 4096 x 12288, 6 bits: 10.6 us for
// 132 MB, 12 TB/s). AHEAD: all loads of a piece are on their way before its
// first product; left alone they alternate with the products in fewer registers. It pays with fewer than 8
// waves a CU (64 x 4096 x 12288: 12.1 us with, 15.8 without) and costs above (256 x 4096 x 4096: 11.3 with, 10.4 without).
template <int TYPE, int G, int RT, int TT, int NW, bool FQ, bool AHEAD>
__global__ __launch_bounds__(64 * NW) void kq4_mx_rows_kernel(KQ4MxArgs a, int ks, int mtiles, int all, int turn) {
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  constexpr int W = G * RT;                              // weight tiles of a wave: [matrix][row tile]
  // XCD x works on a run of row tiles, each against all tokens before the next: its cache reads the weights once; or
  // (turn: the row tiles' workgroups) on a run of tokens against all rows, and reads the activations once
  const int xcd = blockIdx.x & 7, q8 = all >> 3, r8 = all & 7;
  const int v = xcd * q8 + (xcd < r8 ? xcd : r8) + (int)(blockIdx.x >> 3);
  const int tw = turn ? v % turn : v / mtiles, m0 = (turn ? v / turn : v % mtiles) * TT;
  const int t = (tw * (NW / ks) + wave / ks) * RT, slice = wave % ks;
  const KQ4MxDims dw = kq4_mx_dims(a.rows, a.cols), dx = kq4_mx_dims(a.n, a.cols);
  uint32_t wstep[W];   // from a tile to the next, in tiles (a row tile's offsets stay below 2^32: cols <= 2^20)
  const uint8_t *w[W], *ws[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int tc = min(t + i % RT, dw.nt - 1);           // past the last tile: that one again, not stored
    wstep[i] = (uint32_t)kq4_mx_step(tc, dw.nt);
    w[i] = a.w[i / RT] + kq4_mx_first(tc, dw.kt) * 1024;
    ws[i] = a.w[i / RT] + kq4_mx_codes_size(dw, 4) + kq4_mx_first(tc, dw.kq) * KQ4_MX_STILE;
  }
  const int nq = dw.kq, last = dw.kt - 1;

  // FQ: [token][block] codes (their first 16 bytes, then the rest of all), then [token][512 columns][4] scale dwords
  const int nb = 4 * dw.kt, nbs = 16 * nq, real = a.cols >> 5;   // blocks of a token: with codes, with scales, with values
  const int nt = min(16 * TT, a.n - 16 * m0);                    // the workgroup's tokens
  uint8_t *xc = lds, *xr = lds + (size_t)nt * nb * 16, *xsc = xr + (TYPE == 6 ? (size_t)nt * nb * 8 : 0);
  float4 fx[8];
  auto fetch = [&](int e) {
    const int t = e / nbs, b = min(e - t * nbs, real - 1);       // (a block past the columns: the last one, not used)
    const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.x) +
                                                       (size_t)(16 * m0 + min(t, nt - 1)) * a.ldx + 32 * b);
#pragma unroll
    for (int i = 0; i < 8; ++i) fx[i] = p[i];
  };
  auto quantize = [&](int e) {
    const int t = e / nbs, b = e - t * nbs;
    uint32_t s = 0, o[TYPE] = {};
    if (b < real) {
      float v[32];
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[4 * i] = fx[i].x; v[4 * i + 1] = fx[i].y; v[4 * i + 2] = fx[i].z; v[4 * i + 3] = fx[i].w;
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) m = max(m, kq4_absbits(v[i]));
      s = kq4_mx_scale_byte(m, TYPE);
      kq4_mx_encode<TYPE>(v, s, o);
    }
    if (b < nb) {
      *reinterpret_cast<uint4 *>(xc + ((size_t)t * nb + b) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
      if constexpr (TYPE == 6) *reinterpret_cast<uint2 *>(xr + ((size_t)t * nb + b) * 8) = make_uint2(o[4], o[5]);
    }
    xsc[((size_t)t * nq + (b >> 4)) * 16 + 4 * (b & 3) + ((b >> 2) & 3)] = (uint8_t)s;
  };
  const uint8_t *x[TT], *xs[TT];
  uint32_t xstep[TT];
  if constexpr (!FQ) {
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int u = min(m0 + i, dx.nt - 1);
      xstep[i] = (uint32_t)kq4_mx_step(u, dx.nt);
      x[i] = static_cast<const uint8_t *>(a.x) + kq4_mx_first(u, dx.kt) * (256 * TYPE);
      xs[i] = static_cast<const uint8_t *>(a.x) + kq4_mx_codes_size(dx, TYPE) + kq4_mx_first(u, dx.kq) * KQ4_MX_STILE;
    }
  }

  // (past the last column tile: that one again; its scales there are 2^-127 on both sides, so it adds nothing)
  struct Acts {
    uint4 c[4][TT];
    uint2 r[4][TT];
    uint32_t s[TT];
  };
  auto load_x = [&](Acts &p, int q) {
#pragma unroll
    for (int j = 0; j < TT; ++j) {
      const int tok = min(16 * j + r16, nt - 1);         // FQ: lanes past the tokens repeat the last one
      if constexpr (FQ) p.s[j] = *reinterpret_cast<const uint32_t *>(xsc + ((size_t)tok * nq + q) * 16 + 4 * g4);
      else p.s[j] = reinterpret_cast<const uint32_t *>(xs[j] + (uint32_t)q * (xstep[j] * KQ4_MX_STILE))[lane];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int k = min(4 * q + s, last);
        p.r[s][j] = make_uint2(0u, 0u);
        if constexpr (FQ) {
          const size_t b = (size_t)tok * nb + 4 * k + g4;
          p.c[s][j] = *reinterpret_cast<const uint4 *>(xc + b * 16);
          if constexpr (TYPE == 6) p.r[s][j] = *reinterpret_cast<const uint2 *>(xr + b * 8);
        } else {
          const uint8_t *c = x[j] + (uint32_t)k * (xstep[j] * (256 * TYPE));
          p.c[s][j] = reinterpret_cast<const uint4 *>(c)[lane];
          if constexpr (TYPE == 6) p.r[s][j] = reinterpret_cast<const uint2 *>(c + 1024)[lane];
        }
      }
    }
  };
  struct Weights {
    kq4_v4u c[W][4];
    uint32_t s[W];
  };
  auto load_w = [&](Weights &p, int q) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint32_t *sp = reinterpret_cast<const uint32_t *>(ws[i] + (uint32_t)q * (wstep[i] * KQ4_MX_STILE)) + lane;
      p.s[i] = TT == 1 ? __builtin_nontemporal_load(sp) : *sp;   // (with more tokens other workgroups read them too)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const kq4_v4u *cp =
            reinterpret_cast<const kq4_v4u *>(w[i] + (uint32_t)min(4 * q + j, last) * (wstep[i] * 1024)) + lane;
        p.c[i][j] = TT == 1 ? __builtin_nontemporal_load(cp) : *cp;
      }
    }
  };
  kq4_v4f acc[W][TT];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = kq4_v4f{0.0f, 0.0f, 0.0f, 0.0f};
  auto products = [&](const Weights &p, const Acts &y) {
    kq4_v8i xv[4][TT];
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int j = 0; j < TT; ++j)
        xv[s][j] = kq4_v8i{(int)y.c[s][j].x, (int)y.c[s][j].y, (int)y.c[s][j].z, (int)y.c[s][j].w,
                           (int)y.r[s][j].x, (int)y.r[s][j].y, 0, 0};
#define KQ4_MX_STEP(S)                                                                                               \
  _Pragma("unroll") for (int i = 0; i < W; ++i) {                                                                    \
    const kq4_v8i wv = {(int)p.c[i][S].x, (int)p.c[i][S].y, (int)p.c[i][S].z, (int)p.c[i][S].w, 0, 0, 0, 0};         \
    _Pragma("unroll") for (int j = 0; j < TT; ++j) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(     \
        wv, xv[S][j], acc[i][j], 4, kq4_mx_fmt<TYPE>, S, (int)p.s[i], S, (int)y.s[j]);                               \
  }
    KQ4_MX_STEP(0)
    KQ4_MX_STEP(1)
    KQ4_MX_STEP(2)
    KQ4_MX_STEP(3)
#undef KQ4_MX_STEP
  };
  Weights pw;
  if constexpr (FQ) {
    fetch(threadIdx.x);
    load_w(pw, min(slice, nq - 1));
    for (int e = threadIdx.x; e < nt * nbs; e += 64 * NW) {
      if (e >= 64 * NW) fetch(e);
      quantize(e);
    }
    __syncthreads();
  }
  for (int q = slice; q < nq; q += ks) {
    Acts px;
    load_x(px, q);
    if (!FQ || q != slice) load_w(pw, q);
    if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
    products(pw, px);
  }

  // lane (token & 15) + 16 * (row >> 2 & 3) holds rows 4 * (row >> 2) .. + 3 of a tile
  if (ks > 1) {   // [wave][weight tile][token tile][lane][4]
    if constexpr (FQ) __syncthreads();   // the activations' LDS is free
    kq4_v4f *red = reinterpret_cast<kq4_v4f *>(lds);
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < TT; ++j) red[((wave * W + i) * TT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // token tile j is added up and stored by the wave of slice j % ks
#pragma unroll
    for (int j = 0; j < TT; ++j)
      if (slice == (j & (ks - 1)))
#pragma unroll
        for (int i = 0; i < W; ++i) {
          acc[i][j] = red[(((wave - slice) * W + i) * TT + j) * 64 + lane];
          for (int v = 1; v < ks; ++v) acc[i][j] += red[(((wave - slice + v) * W + i) * TT + j) * 64 + lane];
        }
  }
  const bool by4 = (((uintptr_t)a.out | (uintptr_t)a.res | (uintptr_t)(a.ldo * 4)) & 15) == 0;   // (the four in one access)
#pragma unroll
  for (int j = 0; j < TT; ++j) {
    const int T = 16 * (m0 + j) + r16;
    if (slice != (j & (ks - 1)) || T >= a.n) continue;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int R = 16 * (t + r) + 4 * g4;
      const size_t at = (size_t)T * a.ldo + R;
      kq4_v4f y = acc[r][j];
      if constexpr (G == 2) y = kq4_mx_gate<4>(y, acc[RT + r][j]);
      if (by4 && R + 4 <= a.rows) {
        if (a.res) y += *reinterpret_cast<const kq4_v4f *>(a.res + at);
        *reinterpret_cast<kq4_v4f *>(a.out + at) = y;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (R + e < a.rows) a.out[at + e] = a.res ? y[e] + a.res[at + e] : y[e];
      }
    }
  }
}

// LDS of the activations that a workgroup quantizes itself.
static size_t kq4_mx_rows_lds(int n, const KQ4MxDims &d, int type) { return (size_t)n * (4 * d.kt * 4 * type + 16 * d.kq); }

template <int TYPE, int G, int RT, int TT, int NW, bool FQ, bool AHEAD>
static int launch(const KQ4MxArgs &a, int ks, hipStream_t s) {
  const KQ4MxDims dw = kq4_mx_dims(a.rows, a.cols), dx = kq4_mx_dims(a.n, a.cols);
  const int tpw = NW / ks * RT, mtiles = (dx.nt + TT - 1) / TT, all = (dw.nt + tpw - 1) / tpw * mtiles;
  // Tokens outside where the activations are more than the weights and than an XCD's cache of 4 MB: 4096 x 256 x 12288, 6 bits,
  // 21 us so and 45 with the rows outside; 512 x 128 x 4096 4.5 and 4.0.
  const size_t xs = kq4_mx_size(dx, TYPE);
  const bool turn = xs > (4u << 20) && xs > G * kq4_mx_size(dw, 4);
  const size_t red = ks > 1 ? (size_t)NW * G * RT * TT * 1024 : 0, x = FQ ? kq4_mx_rows_lds(min(a.n, 16 * TT), dw, TYPE) : 0;
  hipLaunchKernelGGL((kq4_mx_rows_kernel<TYPE, G, RT, TT, NW, FQ, AHEAD>), dim3((unsigned)all), dim3(64 * NW), red > x ? red : x, s,
                     a, ks, mtiles, all, turn ? all / mtiles : 0);
  return (int)hipGetLastError();
}

// The waves that share a row tile: 8 (a workgroup) where K has that many pieces and the launch then is at most 8 waves a
// CU, else 4 or as many as there are pieces, in workgroups of 4 waves. One token: 4096 x 4096 4.4 us with 8 and 4.9 with 4,
// 12288 x 4096 8.2 and 7.0, 151936 x 2048 51 and 26.
static int slices(const KQ4MxDims &dw, long tiles, int ncu) {
  if (dw.kq >= 8 && tiles <= ncu) return 8;
  int ks = 4;
  while (ks > dw.kq) ks /= 2;
  return ks;
}

// The same where the workgroups quantize the activations: past a tile a CU, workgroups of 8 waves and as many slices as
// leave one workgroup a CU, so that few of them repeat that work (151936 x 2048, three tokens: 28.8 us with 8 waves of a
// tile each, 40.8 with 4 waves on a tile; 50000 x 1024, one token: 6.6 and 10.3; but 12288 x 4096, one token: 7.7 and 7.3).
static int fused_slices(const KQ4MxDims &dw, long tiles, int ncu, int &waves) {
  waves = 8;
  if (tiles <= ncu) {
    const int ks = slices(dw, tiles, ncu);
    if (ks < 8) waves = 4;
    return ks;
  }
  int ks = 4;
  while (ks > 1 && (ks > dw.kq || tiles * ks > 8L * ncu)) ks /= 2;
  return ks;
}

// FEW, MANY: launches of at most a tile a CU, and of 8 waves a CU and more, come here.
template <int TYPE, int G, int RT, int TT, bool FEW, bool MANY>
static int launch_k(const KQ4MxArgs &a, int ncu, hipStream_t s) {
  const KQ4MxDims dw = kq4_mx_dims(a.rows, a.cols), dx = kq4_mx_dims(a.n, a.cols);
  const long tiles = (long)((dw.nt + RT - 1) / RT) * ((dx.nt + TT - 1) / TT);
  const int ks = slices(dw, tiles, ncu);
  if constexpr (FEW)
    if (ks == 8) return launch<TYPE, G, RT, TT, 8, false, true>(a, ks, s);
  if constexpr (MANY)
    if (tiles * ks >= 8L * ncu) return launch<TYPE, G, RT, TT, 4, false, false>(a, ks, s);
  return launch<TYPE, G, RT, TT, 4, false, true>(a, ks, s);
}

template <int TYPE, int G>
static int launch_fused(const KQ4MxArgs &a, int ncu, hipStream_t s) {
  const KQ4MxDims dw = kq4_mx_dims(a.rows, a.cols);
  int waves;
  const int ks = fused_slices(dw, (long)dw.nt * ((a.n + 15) / 16), ncu, waves);
  return waves == 8 ? launch<TYPE, G, 1, 1, 8, true, false>(a, ks, s) : launch<TYPE, G, 1, 1, 4, true, false>(a, ks, s);
}

// A wave's tile: the smallest with at most 1.75 tiles a CU, as few waves cover a piece's latency badly (128 x 1024 x 1024, 6
// bits: 3.0 us with 16 rows x 16 tokens, 4.3 with 32 x 32); else the largest, which loads the least (128 x 4096 x 12288: 14.2 with
// 32 x 64, 19.2 with 32 x 32; 64 x 32 is as good: better at 6 bits, worse at 4). One tile of tokens where there are 16 or 32
// of them, of 32 rows where rows are many (16 x 151936 x 2048: 30.7 us, of 16 rows 34.8; 32 tokens 41.2 and 49.9; but 16 x
// 12288 x 4096 8.6 and 8.1). Within 2.8 % of the best of six tiles (17 to 300 tokens of nine matrices).
template <int TYPE, int G>
static int launch_t(const KQ4MxArgs &a, int ncu, hipStream_t s) {
  if (a.ldx) return launch_fused<TYPE, G>(a, ncu, s);
  const KQ4MxDims dw = kq4_mx_dims(a.rows, a.cols), dx = kq4_mx_dims(a.n, a.cols);
  auto few = [&](int rt, int tt) { return 4L * ((dw.nt + rt - 1) / rt) * ((dx.nt + tt - 1) / tt) <= 7L * ncu; };
  if constexpr (G == 1)
    if (a.n <= 16 && dw.nt > 4 * ncu) return launch_k<TYPE, G, 2, 1, false, true>(a, ncu, s);
  if (a.n <= 16 || few(1, 1)) return launch_k<TYPE, G, 1, 1, true, true>(a, ncu, s);
  if (few(1, 2) || (G == 2 && a.n <= 32)) return launch_k<TYPE, G, 1, 2, true, G == 2>(a, ncu, s);
  if constexpr (G == 2) return launch_k<TYPE, G, 1, 4, true, true>(a, ncu, s);
  else if (a.n <= 32 || few(2, 2)) return launch_k<TYPE, G, 2, 2, true, true>(a, ncu, s);
  else return launch_k<TYPE, G, 2, 4, true, true>(a, ncu, s);
}

int kq4_launch_mx_rows(const KQ4MxArgs &a, int type, int ncu, hipStream_t s) {
  if (a.w[1]) return type == 4 ? launch_t<4, 2>(a, ncu, s) : launch_t<6, 2>(a, ncu, s);
  return type == 4 ? launch_t<4, 1>(a, ncu, s) : launch_t<6, 1>(a, ncu, s);
}

// Every workgroup quantizes its tokens' activations, 0.12 us for 1000 elements of each workgroup that its CU runs, against a
// launch of the quantizer (2.5 to 3.4 us, and as much of the host's time). Worth it up to 24576 elements a CU, up to 32768 in
// launches of a tile a CU, where the host takes the longer (4096 x 4096: four tokens 6.1 us against 7.4, eight 8.1 against 7.5
// and a launch less, sixteen 11.8 against 7.5; 12288 x 4096, eight tokens: 11.2 against 10.4), up to 8192 where more tokens
// have wider tiles without it (32 x 4096 x 512: 4.5 against 6.4; 32 x 6144 x 2048: 9.1 against 7.7), and where the weights
// take the memory longer than that anyway (151936 x 2048: one token 27 us against 31, four 28 and 30, eight 32 and 30.5).
bool kq4_mx_rows_fused(int n, int rows, int cols, int matrices, int type, int ncu) {
  const KQ4MxDims d = kq4_mx_dims(rows, cols);
  const int tokens = min(n, 16), mtiles = (n + 15) / 16;
  const long tiles = (long)d.nt * mtiles;
  if (kq4_mx_rows_lds(tokens, d, type) > 64 * 1024) return false;
  int waves;
  const int ks = fused_slices(d, tiles, ncu, waves), tpw = waves / ks;
  const double wgs = (double)((d.nt + tpw - 1) / tpw) * mtiles, each = (wgs > ncu ? wgs / ncu : 1.0) * tokens * cols;
  return each <= (tiles <= ncu ? 32768.0 : n <= 16 ? 24576.0 : 8192.0) ||
         (n <= 16 && each * 0.12e-3 <= 0.3 * matrices * rows * (double)cols * 0.53 / 6.0e6);
}
