// kq4_mx_rows.hip - products of few tokens with 4-bit microscaled weights.
//   out[t][r] = [res[t][r] +] sum_k x[t][k] w[r][k]                    (G = 1)
//   out[t][r] = silu(sum_k x[t][k] wg[r][k]) * sum_k x[t][k] wu[r][k]  (G = 2)
#include "kq4_internal.h"
#include "kq4_mx_dev.h"

#define KQ4_MXR_WAVES 8

// A wave takes a row tile of 16 rows (of each matrix) against 16 * TT tokens and every KS-th piece of 512 columns (a
// dword of scales per lane, a byte for each 128 of them); KS waves of a workgroup share a row tile, and their sums are
// added in LDS in wave order. The weights, read once, go from memory to the registers of
// v_mfma_scale_f32_16x16x128_f8f6f4 as they lie, a tile one 16-byte load per lane, D pieces on their way at a time.
// The activations come the same way from a quantized matrix (FQ = 0), or the workgroup quantizes the fp32 rows into LDS
// while its first weights are on their way (FQ = 1): one launch instead of two.
template <int TYPE, int G, int TT, int D, bool FQ>
__global__ __launch_bounds__(64 * KQ4_MXR_WAVES) void kq4_mx_rows_kernel(KQ4MxArgs a, int ks) {
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  const int tpw = KQ4_MXR_WAVES / ks;                    // row tiles of the workgroup
  const int t = (int)blockIdx.x * tpw + wave / ks, slice = wave % ks, m0 = (int)blockIdx.y * TT;
  const KQ4MxDims dw = a.dw, dx = a.dx;
  const int tc = min(t, dw.nt - 1);                      // past the last tile: that one again, not stored
  const long wstep = kq4_mx_step(tc, dw.nt);
  const uint8_t *w[G], *ws[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    w[g] = a.w[g] + kq4_mx_first(tc, dw.kt) * 1024;
    ws[g] = a.w[g] + kq4_mx_codes_size(dw, 4) + kq4_mx_first(tc, dw.kq) * KQ4_MX_STILE;
  }
  const int nq = dw.kq, last = dw.kt - 1;
  struct Piece {
    kq4_v4u c[G][4];
    uint32_t s[G];
  } pw[D];
  // (past the last column tile: that one again; its scales there are 2^-127 on both sides, so it adds nothing)
  auto load = [&](Piece &p, int q) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      p.s[g] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(ws[g] + q * wstep * KQ4_MX_STILE) + lane);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p.c[g][j] = __builtin_nontemporal_load(
            reinterpret_cast<const kq4_v4u *>(w[g] + min(4 * q + j, last) * wstep * 1024) + lane);
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(pw[d], min(slice + d * ks, nq - 1));

  // FQ: [token][block] codes (their first 16 bytes, then the rest of all), then [token][512 columns][4] scale dwords
  const int nb = 4 * dw.kt;
  uint8_t *xc = lds, *xr = lds + (size_t)a.n * nb * 16, *xsc = xr + (TYPE == 6 ? (size_t)a.n * nb * 8 : 0);
  if constexpr (FQ) {
    const int nbs = 16 * nq, real = a.cols >> 5;         // blocks of a token: with scales, with values
    for (int e = threadIdx.x; e < a.n * nbs; e += blockDim.x) {
      const int tok = e / nbs, b = e - tok * nbs;
      uint32_t s = 0, o[TYPE] = {};
      if (b < real) {
        float v[32];
        const float4 *p = reinterpret_cast<const float4 *>(a.xf + (size_t)tok * a.ldx + 32 * b);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 f = p[i];
          v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) m = max(m, kq4_absbits(v[i]));
        s = kq4_mx_scale_byte(m, TYPE);
        kq4_mx_encode<TYPE>(v, s, o);
      }
      if (b < nb) {
        *reinterpret_cast<uint4 *>(xc + ((size_t)tok * nb + b) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
        if constexpr (TYPE == 6) *reinterpret_cast<uint2 *>(xr + ((size_t)tok * nb + b) * 8) = make_uint2(o[4], o[5]);
      }
      xsc[((size_t)tok * nq + (b >> 4)) * 16 + 4 * (b & 3) + ((b >> 2) & 3)] = (uint8_t)s;
    }
    __syncthreads();
  }
  const uint8_t *x[TT], *xs[TT];
  long xstep[TT];
  if constexpr (!FQ) {
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int u = min(m0 + i, dx.nt - 1);
      xstep[i] = kq4_mx_step(u, dx.nt);
      x[i] = a.x + kq4_mx_first(u, dx.kt) * (256 * TYPE);
      xs[i] = a.x + kq4_mx_codes_size(dx, TYPE) + kq4_mx_first(u, dx.kq) * KQ4_MX_STILE;
    }
  }
  const int tok = min(r16, a.n - 1);                     // FQ: lanes past the tokens repeat the last one

  kq4_v4f acc[G][TT];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[g][j] = kq4_v4f{0.0f, 0.0f, 0.0f, 0.0f};
  auto products = [&](const Piece &p, int q) {
    uint32_t sx[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) {
      if constexpr (FQ) sx[j] = *reinterpret_cast<const uint32_t *>(xsc + ((size_t)tok * nq + q) * 16 + 4 * g4);
      else sx[j] = reinterpret_cast<const uint32_t *>(xs[j] + q * xstep[j] * KQ4_MX_STILE)[lane];
    }
    kq4_v8i xv[4][TT];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = min(4 * q + s, last);
#pragma unroll
      for (int j = 0; j < TT; ++j) {
        uint4 v;
        uint2 u = make_uint2(0u, 0u);
        if constexpr (FQ) {
          const size_t b = (size_t)tok * nb + 4 * k + g4;
          v = *reinterpret_cast<const uint4 *>(xc + b * 16);
          if constexpr (TYPE == 6) u = *reinterpret_cast<const uint2 *>(xr + b * 8);
        } else {
          const uint8_t *c = x[j] + k * xstep[j] * (256 * TYPE);
          v = reinterpret_cast<const uint4 *>(c)[lane];
          if constexpr (TYPE == 6) u = reinterpret_cast<const uint2 *>(c + 1024)[lane];
        }
        xv[s][j] = kq4_v8i{(int)v.x, (int)v.y, (int)v.z, (int)v.w, (int)u.x, (int)u.y, 0, 0};
      }
    }
#define KQ4_MX_STEP(S)                                                                                               \
  _Pragma("unroll") for (int g = 0; g < G; ++g) {                                                                    \
    const kq4_v8i wv = {(int)p.c[g][S].x, (int)p.c[g][S].y, (int)p.c[g][S].z, (int)p.c[g][S].w, 0, 0, 0, 0};         \
    _Pragma("unroll") for (int j = 0; j < TT; ++j) acc[g][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(     \
        wv, xv[S][j], acc[g][j], 4, kq4_mx_fmt<TYPE>, S, (int)p.s[g], S, (int)sx[j]);                                \
  }
    KQ4_MX_STEP(0)
    KQ4_MX_STEP(1)
    KQ4_MX_STEP(2)
    KQ4_MX_STEP(3)
#undef KQ4_MX_STEP
  };
  for (int q = slice; q < nq; q += D * ks) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (q + d * ks < nq) products(pw[d], q + d * ks);
      if (q + D * ks < nq) load(pw[d], min(q + (D + d) * ks, nq - 1));
    }
  }

  // lane (token & 15) + 16 * (row >> 2 & 3) holds rows 4 * (row >> 2) .. + 3 of a tile
  if (ks > 1) {   // [wave][g][j][lane][4]
    if constexpr (FQ) __syncthreads();   // the activations' LDS is free
    kq4_v4f *red = reinterpret_cast<kq4_v4f *>(lds);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < TT; ++j) red[((wave * G + g) * TT + j) * 64 + lane] = acc[g][j];
    __syncthreads();
    if (slice == 0)
      for (int v = 1; v < ks; ++v)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int j = 0; j < TT; ++j) acc[g][j] += red[(((wave + v) * G + g) * TT + j) * 64 + lane];
  }
  if (slice != 0 || t >= dw.nt) return;
#pragma unroll
  for (int j = 0; j < TT; ++j) {
    const int T = 16 * (m0 + j) + r16;
    if (T >= a.n) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int R = 16 * t + 4 * g4 + i;
      if (R >= a.rows) continue;
      float y = acc[0][j][i];
      if constexpr (G == 2) y = kq4_mx_gate(y, acc[1][j][i]);
      const size_t at = (size_t)T * a.ldo + R;
      a.out[at] = a.res ? y + a.res[at] : y;
    }
  }
}

template <int TYPE, int G, int TT, int D, bool FQ>
static int launch(const KQ4MxArgs &a, int ks, hipStream_t s) {
  const int tpw = KQ4_MXR_WAVES / ks;
  const dim3 grid((a.dw.nt + tpw - 1) / tpw, FQ ? 1 : (a.dx.nt + TT - 1) / TT);
  const size_t red = ks > 1 ? (size_t)KQ4_MXR_WAVES * G * TT * 1024 : 0, x = FQ ? kq4_mx_rows_lds(a.n, a.dw, TYPE) : 0;
  hipLaunchKernelGGL((kq4_mx_rows_kernel<TYPE, G, TT, D, FQ>), grid, dim3(64 * KQ4_MXR_WAVES), red > x ? red : x, s, a, ks);
  return (int)hipGetLastError();
}

size_t kq4_mx_rows_lds(int n, const KQ4MxDims &d, int type) { return (size_t)n * (4 * d.kt * 4 * type + 16 * d.kq); }

template <int TYPE, int G, int TT, bool FQ>
static int launch_d(const KQ4MxArgs &a, int ks, hipStream_t s) {
  const int pieces = (a.dw.kq + ks - 1) / ks;
  if (pieces == 1) return launch<TYPE, G, TT, 1, FQ>(a, ks, s);
  if (pieces == 2) return launch<TYPE, G, TT, 2, FQ>(a, ks, s);
  return launch<TYPE, G, TT, 3, FQ>(a, ks, s);
}

template <int TYPE, int G>
static int launch_t(const KQ4MxArgs &a, int ks, hipStream_t s) {
  if (a.xf) return launch_d<TYPE, G, 1, true>(a, ks, s);
  if (a.n <= 16) return launch_d<TYPE, G, 1, false>(a, ks, s);
  return launch_d<TYPE, G, 2, false>(a, ks, s);
}

int kq4_launch_mx_rows(const KQ4MxArgs &a, int type, int ncu, hipStream_t s) {
  int ks = 1;
  while (ks < KQ4_MXR_WAVES && 2 * ks <= a.dw.kq && (long)a.dw.nt * ks < 8L * ncu) ks *= 2;
  if (a.w[1]) return type == 4 ? launch_t<4, 2>(a, ks, s) : launch_t<6, 2>(a, ks, s);
  return type == 4 ? launch_t<4, 1>(a, ks, s) : launch_t<6, 1>(a, ks, s);
}
