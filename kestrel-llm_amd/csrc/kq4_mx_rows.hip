// kq4_mx_rows.hip - products of few tokens with 4-bit microscaled weights.
//   out[t][r] = [res[t][r] +] sum_k x[t][k] w[r][k]                    (G = 1)
//   out[t][r] = silu(sum_k x[t][k] wg[r][k]) * sum_k x[t][k] wu[r][k]  (G = 2)
#include "kq4_internal.h"
#include "kq4_mx_dev.h"

// A workgroup takes 16 * RT rows of the weights against 16 * TT tokens and deals K to its waves in pieces of 512
// columns (one dword of scales per lane, a byte for each 128). Weights and activations go from memory to the registers
// of v_mfma_scale_f32_16x16x128_f8f6f4 as they lie: a tile is one 16-byte load per lane (and one of 8 bytes for 6-bit activations).
// The waves' sums are added in LDS in wave order.
template <int TYPE, int G, int RT, int TT>
__global__ __launch_bounds__(512) void kq4_mx_rows_kernel(KQ4MxArgs a) {
  extern __shared__ __align__(16) float red[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int t0 = blockIdx.x * RT, m0 = blockIdx.y * TT;
  const KQ4MxDims dw = a.dw, dx = a.dx;
  const uint8_t *w[G][RT], *ws[G][RT], *x[TT], *xs[TT];
  long wstep[RT], xstep[TT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int t = min(t0 + i, dw.nt - 1);   // past the last tile: that one again, not stored
    wstep[i] = kq4_mx_step(t, dw.nt);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      w[g][i] = a.w[g] + kq4_mx_first(t, dw.kt) * 1024 + 16 * lane;
      ws[g][i] = a.w[g] + kq4_mx_codes_size(dw, 4) + kq4_mx_first(t, dw.kq) * KQ4_MX_STILE + 4 * lane;
    }
  }
#pragma unroll
  for (int i = 0; i < TT; ++i) {
    const int t = min(m0 + i, dx.nt - 1);
    xstep[i] = kq4_mx_step(t, dx.nt);
    x[i] = a.x + kq4_mx_first(t, dx.kt) * (256 * TYPE);
    xs[i] = a.x + kq4_mx_codes_size(dx, TYPE) + kq4_mx_first(t, dx.kq) * KQ4_MX_STILE + 4 * lane;
  }
  kq4_v4f acc[G][RT][TT];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < TT; ++j) acc[g][i][j] = kq4_v4f{0.0f, 0.0f, 0.0f, 0.0f};
  for (int q = wave; q < dw.kq; q += nw) {
    uint32_t sw[G][RT], sx[TT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int g = 0; g < G; ++g) sw[g][i] = *reinterpret_cast<const uint32_t *>(ws[g][i] + q * wstep[i] * KQ4_MX_STILE);
#pragma unroll
    for (int j = 0; j < TT; ++j) sx[j] = *reinterpret_cast<const uint32_t *>(xs[j] + q * xstep[j] * KQ4_MX_STILE);
#define KQ4_MX_STEP(S)                                                                                            \
  if (4 * q + S < dw.kt) {                                                                                        \
    const long k = 4 * q + S;                                                                                     \
    kq4_v8i wv[G][RT], xv[TT];                                                                                    \
    _Pragma("unroll") for (int g = 0; g < G; ++g) _Pragma("unroll") for (int i = 0; i < RT; ++i) {                \
      const uint4 v = *reinterpret_cast<const uint4 *>(w[g][i] + k * wstep[i] * 1024);                            \
      wv[g][i] = kq4_v8i{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};                                     \
    }                                                                                                             \
    _Pragma("unroll") for (int j = 0; j < TT; ++j) {                                                              \
      const uint8_t *p = x[j] + k * xstep[j] * (256 * TYPE);                                                      \
      const uint4 v = *reinterpret_cast<const uint4 *>(p + 16 * lane);                                            \
      uint2 u = make_uint2(0u, 0u);                                                                               \
      if constexpr (TYPE == 6) u = *reinterpret_cast<const uint2 *>(p + 1024 + 8 * lane);                         \
      xv[j] = kq4_v8i{(int)v.x, (int)v.y, (int)v.z, (int)v.w, (int)u.x, (int)u.y, 0, 0};                          \
    }                                                                                                             \
    _Pragma("unroll") for (int g = 0; g < G; ++g) _Pragma("unroll") for (int i = 0; i < RT; ++i)                  \
        _Pragma("unroll") for (int j = 0; j < TT; ++j) acc[g][i][j] =                                             \
            __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv[g][i], xv[j], acc[g][i][j], 4, kq4_mx_fmt<TYPE>,  \
                                                             S, (int)sw[g][i], S, (int)sx[j]);                    \
  }
    KQ4_MX_STEP(0)
    KQ4_MX_STEP(1)
    KQ4_MX_STEP(2)
    KQ4_MX_STEP(3)
#undef KQ4_MX_STEP
  }
  // lane (token & 15) + 16 * (row >> 2 & 3) holds rows 4 * (row >> 2) .. + 3 of a tile: [wave][g][i][j][lane][4]
  constexpr int NA = G * RT * TT;
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < TT; ++j)
        *reinterpret_cast<kq4_v4f *>(&red[((wave * NA + (g * RT + i) * TT + j) * 64 + lane) * 4]) = acc[g][i][j];
  __syncthreads();
  for (int e = threadIdx.x; e < RT * TT * 256; e += blockDim.x) {
    const int row = e % (16 * RT), tok = e / (16 * RT), i = row >> 4, j = tok >> 4;
    const int at = ((tok & 15) + 16 * ((row >> 2) & 3)) * 4 + (row & 3);
    float s[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      s[g] = 0.0f;
      for (int v = 0; v < nw; ++v) s[g] += red[(v * NA + (g * RT + i) * TT + j) * 256 + at];
    }
    const int R = 16 * t0 + row, T = 16 * m0 + tok;
    if (R < a.rows && T < a.n) {
      float y = s[0];
      if constexpr (G == 2) y = kq4_mx_gate(s[0], s[1]);
      if (a.res) y += a.res[(size_t)T * a.ldo + R];
      a.out[(size_t)T * a.ldo + R] = y;
    }
  }
}

template <int TYPE, int G, int RT, int TT>
static int launch(const KQ4MxArgs &a, hipStream_t s) {
  const int nw = a.dw.kq < 8 ? a.dw.kq : 8;
  const dim3 grid((a.dw.nt + RT - 1) / RT, (a.dx.nt + TT - 1) / TT);
  hipLaunchKernelGGL((kq4_mx_rows_kernel<TYPE, G, RT, TT>), grid, dim3(64 * nw), nw * G * RT * TT * 1024, s, a);
  return (int)hipGetLastError();
}

int kq4_launch_mx_rows(const KQ4MxArgs &a, int type, hipStream_t s) {
  if (a.w[1]) return type == 4 ? launch<4, 2, 1, 1>(a, s) : launch<6, 2, 1, 1>(a, s);
  return type == 4 ? launch<4, 1, 1, 2>(a, s) : launch<6, 1, 1, 2>(a, s);
}
