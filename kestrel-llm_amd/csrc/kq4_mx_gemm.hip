// kq4_mx_gemm.hip - products of many tokens with 4-bit microscaled weights (the sums of kq4_mx_rows.hip).
#include "kq4_internal.h"
#include "kq4_mx_dev.h"

// A workgroup takes 64 WM tokens x 128 WN rows (gated: 64 WN rows of each projection), a wave 64 x 128 of it: 2 x 4
// tiles of v_mfma_scale_f32_32x32x64_f8f6f4, tokens as the first operand, so that an accumulator register is 32
// consecutive outputs of two tokens. A stage is 128 columns; both operands' tiles go from memory straight to LDS, in
// runs of 1 KB as they lie (a group's 8 row tiles are one run), and from there by conflict-free 16-byte reads into the
// matrix unit. The ring holds S stages; a barrier per stage frees the slot that the loads of the stage S - 1 ahead
// go to. Scales of four stages at a time go the same way, then into registers, a byte per stage.
template <int TYPE, int WM, int WN, int S>
struct KQ4MxTile {
  static constexpr int NW = WM * WN, BM = 64 * WM, BN = 128 * WN;
  static constexpr int TA = 256 * TYPE;                       // bytes of an activation tile (16 x 128)
  static constexpr int A = BM / 16 * TA, B = BN / 16 * 1024;  // a stage's operands
  static constexpr int STAGE = A + B, LOADS = STAGE / 1024;
  static constexpr int LPW = (LOADS + NW - 1) / NW;           // loads of a wave per stage
  static constexpr int SCALES = (BM + BN) / 16 * KQ4_MX_STILE, SLOADS = SCALES / 1024;
  static constexpr int SPW = (SLOADS + NW - 1) / NW;
  static constexpr int LDS = S * STAGE + SCALES;
};

template <int TYPE, int G, int WM, int WN, int S, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void kq4_mx_gemm_kernel(KQ4MxArgs a, int mtiles, int ntiles) {
  using T = KQ4MxTile<TYPE, WM, WN, S>;
  constexpr int RG = T::BN / G;                 // output rows of the workgroup
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM, l32 = lane & 31, half = lane >> 5;

  // XCD x works on a run of tiles, in bands of 8 tiles of tokens, so that what it reads at a time is shared
  const int ntile = mtiles * ntiles, xcd = blockIdx.x & 7, q8 = ntile >> 3, r8 = ntile & 7;
  const int v = xcd * q8 + (xcd < r8 ? xcd : r8) + (int)(blockIdx.x >> 3);
  const int band = v / (8 * ntiles), bm = min(8, mtiles - 8 * band), u = v - band * 8 * ntiles;
  const int m0 = (8 * band + u % bm) * T::BM, n0 = (u / bm) * RG;

  // this wave's loads: where each 1-KB run of a stage starts and how far the next stage's lies
  const KQ4MxDims dw = a.dw, dx = a.dx;
  const long xall = (long)kq4_mx_size(dx, TYPE), wall = (long)kq4_mx_size(dw, 4);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t *)&lds[0];
  kq4_rsrc4 src[T::LPW], ssrc[T::SPW];
  uint32_t step[T::LPW], sstep[T::SPW];
  auto resource = [](const uint8_t *p, long at, long all) {   // loads at or past `all` read zeros
    const long left = at < all ? all - at : 0;
    return kq4_rsrc_at(p + (at < all ? at : 0), (uint32_t)(left < 0x7fffffffL ? left : 0x7fffffffL), 0);
  };
  auto where = [&](int c, bool scales, kq4_rsrc4 &r, uint32_t &st) {
    // 1-KB run c of the stage's (or the scales') runs; row tiles in groups of 8, a group's run is tile bytes * 8
    const int ta = scales ? KQ4_MX_STILE : T::TA, tb = scales ? KQ4_MX_STILE : 1024;
    const int ca = T::BM / 16 * ta / 1024;
    const int kx = scales ? dx.kq : dx.kt, kw = scales ? dw.kq : dw.kt;
    if (c < ca) {
      const int t = (m0 >> 4) + c * 1024 / (8 * ta) * 8, off = c * 1024 % (8 * ta);
      const int tt = t < dx.nt ? t : 0;
      // (a workgroup of 64 tokens may start inside a group)
      const int in = (tt & 7) * ta;
      const long at = (long)(tt & ~7) * kx * ta + in + off + (scales ? (long)kq4_mx_codes_size(dx, TYPE) : 0);
      r = resource(a.x, t < dx.nt ? at : xall, xall);
      st = (uint32_t)(kq4_mx_step(tt, dx.nt) * ta);
    } else {
      const int b = (c - ca) * 1024, per = RG / 16 * tb;      // bytes of one matrix' rows
      const uint8_t *w = a.w[G == 2 ? b / per : 0];
      const int o = G == 2 ? b % per : b;
      const int t = (n0 >> 4) + o / (8 * tb) * 8, off = o % (8 * tb);
      const int tt = t < dw.nt ? t : 0;
      const int in = (tt & 7) * tb;
      const long at = (long)(tt & ~7) * kw * tb + in + off + (scales ? (long)kq4_mx_codes_size(dw, 4) : 0);
      r = resource(w, t < dw.nt ? at : wall, wall);
      st = (uint32_t)(kq4_mx_step(tt, dw.nt) * tb);
    }
  };
#pragma unroll
  for (int l = 0; l < T::LPW; ++l) where(min(wave * T::LPW + l, T::LOADS - 1), false, src[l], step[l]);
#pragma unroll
  for (int l = 0; l < T::SPW; ++l) where(min(wave * T::SPW + l, T::SLOADS - 1), true, ssrc[l], sstep[l]);
  const uint32_t v16 = 16u * lane;
  auto load = [&](const kq4_rsrc4 &r, uint32_t soff, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(v16), "s"(r),
                 "s"(soff) : "memory", "m0");
  };
  const int nk = dw.kt, nq = dw.kq;
  auto load_stage = [&](int k, int slot) {      // (past the last stage: that one again, never used)
    const uint32_t kk = (uint32_t)min(k, nk - 1);
#pragma unroll
    for (int l = 0; l < T::LPW; ++l)
      load(src[l], kk * step[l], lds0 + slot * T::STAGE + min(wave * T::LPW + l, T::LOADS - 1) * 1024);
  };
  auto load_scales = [&](int q) {
    const uint32_t qq = (uint32_t)min(q, nq - 1);
#pragma unroll
    for (int l = 0; l < T::SPW; ++l)
      load(ssrc[l], qq * sstep[l], lds0 + S * T::STAGE + min(wave * T::SPW + l, T::SLOADS - 1) * 1024);
  };

  kq4_v16f acc[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  // tile of 32 rows: its first row tile in the operand's LDS region
  const int at = 4 * wm;
  auto bt = [&](int j) { return G == 2 ? (j >> 1) * (RG / 16) + 4 * wn + 2 * (j & 1) : 8 * wn + 2 * j; };
  const int frag = (l32 >> 4), r16 = l32 & 15;

  load_scales(0);
#pragma unroll
  for (int s = 0; s < S - 1; ++s) load_stage(s, s);
  int slot = 0;
  uint32_t sa[2][2], sb[4][2];
  auto stage = [&](int k, auto jc) {
    constexpr int J = decltype(jc)::value;
    // this wave's part of the stage has come and its reads of the slot that is refilled next are done
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * T::LPW) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (J == 0) {
      const uint8_t *p = lds + S * T::STAGE;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int o = (2 * s + half) * 64 + 4 * r16;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          sa[i][s] = *reinterpret_cast<const uint32_t *>(p + (at + 2 * i + frag) * KQ4_MX_STILE + o);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sb[j][s] = *reinterpret_cast<const uint32_t *>(p + (T::BM / 16 + bt(j) + frag) * KQ4_MX_STILE + o);
      }
    }
    if constexpr (J == 1) load_scales((k >> 2) + 1);
    load_stage(k + S - 1, slot == 0 ? S - 1 : slot - 1);
    const uint8_t *pa = lds + slot * T::STAGE, *pb = pa + T::A;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      kq4_v8i fa[2], fb[4];
      const int b = 2 * s + half;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t *t = pa + (at + 2 * i + frag) * T::TA;
        const uint4 x = *reinterpret_cast<const uint4 *>(t + kq4_mx_piece(b, r16));
        uint2 y = make_uint2(0u, 0u);
        if constexpr (TYPE == 6) y = *reinterpret_cast<const uint2 *>(t + kq4_mx_rest(b, r16));
        fa[i] = kq4_v8i{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, 0, 0};
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 x = *reinterpret_cast<const uint4 *>(pb + (bt(j) + frag) * 1024 + kq4_mx_piece(b, r16));
        fb[j] = kq4_v8i{(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[i], fb[j], acc[i][j], kq4_mx_fmt<TYPE>, 4, J,
                                                                      (int)sa[i][s], J, (int)sb[j][s]);
    }
    slot = slot + 1 == S ? 0 : slot + 1;
  };
  for (int k = 0; k < nk; k += 4) {
    stage(k, std::integral_constant<int, 0>{});
    if (k + 1 < nk) stage(k + 1, std::integral_constant<int, 1>{});
    if (k + 2 < nk) stage(k + 2, std::integral_constant<int, 2>{});
    if (k + 3 < nk) stage(k + 3, std::integral_constant<int, 3>{});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the loads past the last stage: LDS is not given back before

#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int tok = m0 + 64 * wm + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3);
      if (tok < a.n) {
        float *o = a.out + (size_t)tok * a.ldo;
        const float *res = a.res ? a.res + (size_t)tok * a.ldo : nullptr;
#pragma unroll
        for (int j = 0; j < 4 / G; ++j) {
          const int row = n0 + (G == 2 ? 64 * wn : 128 * wn) + 32 * j + l32;
          if (row < a.rows) {
            float y = acc[i][j][e];
            if constexpr (G == 2) y = kq4_mx_gate(y, acc[i][2 + j][e]);
            if (res) y += res[row];
            o[row] = y;
          }
        }
      }
    }
}

template <int TYPE, int G, int WM, int WN, int S, int OCC>
static int launch(const KQ4MxArgs &a, hipStream_t s) {
  using T = KQ4MxTile<TYPE, WM, WN, S>;
  auto *k = kq4_mx_gemm_kernel<TYPE, G, WM, WN, S, OCC>;
  static std::atomic<unsigned long long> done{0};
  const hipError_t e = kq4_lds_limit_once(reinterpret_cast<const void *>(k), T::LDS, done);
  if (e != hipSuccess) return (int)e;
  const int mt = (a.n + T::BM - 1) / T::BM, nt = (a.rows + T::BN / G - 1) / (T::BN / G);
  hipLaunchKernelGGL(k, dim3((unsigned)mt * nt), dim3(64 * T::NW), T::LDS, s, a, mt, nt);
  return (int)hipGetLastError();
}

int kq4_launch_mx_gemm(const KQ4MxArgs &a, int type, hipStream_t s) {
  if (a.w[1]) return type == 4 ? launch<4, 2, 2, 2, 3, 2>(a, s) : launch<6, 2, 2, 2, 2, 2>(a, s);
  return type == 4 ? launch<4, 1, 2, 2, 3, 2>(a, s) : launch<6, 1, 2, 2, 2, 2>(a, s);
}
