// kq4_mx_gemm.hip - products of many tokens with 4-bit microscaled weights (the sums of kq4_mx_rows.hip).
#include "kq4_internal.h"
#include "kq4_mx_dev.h"

#include <type_traits>

// A workgroup of WM x WN waves takes 32 TI WM tokens x 32 TJ WN rows (gated: half as many of each projection), a wave TI x
// TJ tiles of v_mfma_scale_f32_32x32x64_f8f6f4, tokens as the first operand, so that an accumulator register is 32
// consecutive outputs of two tokens. A stage is 128 columns; both operands' tiles go from memory straight to LDS, in
// runs of 1 KB as they lie (a group's 8 row tiles are one run), and from there by conflict-free 16-byte reads into the
// matrix unit, half a stage (64 columns) ahead of their use. The ring holds S stages. The barrier stands in the middle
// of a stage's products, where every wave has the stage's second half in registers: the stage ahead has come, and the
// slot is refilled at once. Scales of four stages at a time go the same way, then into registers, a byte per stage.
template <int TYPE, int TI, int TJ, int WM, int WN, int S>
struct KQ4MxTile {
  static constexpr int NW = WM * WN, BM = 32 * TI * WM, BN = 32 * TJ * WN;
  static constexpr int TA = 256 * TYPE;                       // bytes of an activation tile (16 x 128)
  static constexpr int A = BM / 16 * TA, B = BN / 16 * 1024;  // a stage's operands
  static constexpr int STAGE = A + B;
  static constexpr int LA = A / 1024 / NW, LB = B / 1024 / NW, LPW = LA + LB;   // a wave's loads
  static constexpr int SCALES = (BM + BN) / 16 * KQ4_MX_STILE, SLOADS = SCALES / 1024;
  static constexpr int SPW = (SLOADS + NW - 1) / NW;
  static constexpr int LDS = S * STAGE + SCALES;
  // a wave's runs lie in one group of 8 row tiles, and (gated) in one matrix
  static_assert(A % (1024 * NW) == 0 && B % (1024 * NW) == 0 && SLOADS % SPW == 0, "kq4_mx_gemm: runs per wave");
  static_assert(8 * TA % (LA * 1024) == 0 && 8 % LB == 0 && BM % 128 == 0 && BN % 256 == 0, "kq4_mx_gemm: groups");
  static_assert(LDS <= 160 * 1024, "kq4_mx_gemm: LDS");
};

// N runs of 1 KB from offset soff of r to LDS address `to` on: one address register for each four, the rest of it in the
// instructions' offset, which counts on both sides.
template <int N>
KQ4_DEV void kq4_mx_load(const kq4_rsrc4 &r, uint32_t v16, uint32_t soff, uint32_t to) {
  if constexpr (N >= 4)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds\n\t"
                 "buffer_load_dwordx4 %1, %2, %3 offen offset:1024 lds\n\tbuffer_load_dwordx4 %1, %2, %3 offen offset:2048 lds\n\t"
                 "buffer_load_dwordx4 %1, %2, %3 offen offset:3072 lds" ::"s"(to), "v"(v16), "s"(r), "s"(soff) : "memory", "m0");
  else if constexpr (N == 3)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds\n\t"
                 "buffer_load_dwordx4 %1, %2, %3 offen offset:1024 lds\n\tbuffer_load_dwordx4 %1, %2, %3 offen offset:2048 lds"
                 ::"s"(to), "v"(v16), "s"(r), "s"(soff) : "memory", "m0");
  else if constexpr (N == 2)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds\n\t"
                 "buffer_load_dwordx4 %1, %2, %3 offen offset:1024 lds" ::"s"(to), "v"(v16), "s"(r), "s"(soff) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(v16), "s"(r),
                 "s"(soff) : "memory", "m0");
  if constexpr (N > 4) kq4_mx_load<N - 4>(r, v16, soff + 4096, to + 4096);
}

template <int TYPE, int G, int TI, int TJ, int WM, int WN, int S, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void kq4_mx_gemm_kernel(KQ4MxArgs a, int mtiles, int ntiles) {
  using T = KQ4MxTile<TYPE, TI, TJ, WM, WN, S>;
  constexpr int RG = T::BN / G;                 // output rows of the workgroup
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM, l32 = lane & 31, half = lane >> 5;

  // XCD x works on a run of tiles, in bands of 8 tiles of tokens, so that what it reads at a time is shared
  const int ntile = mtiles * ntiles, xcd = blockIdx.x & 7, q8 = ntile >> 3, r8 = ntile & 7;
  const int v = xcd * q8 + (xcd < r8 ? xcd : r8) + (int)(blockIdx.x >> 3);
  const int band = v / (8 * ntiles), bm = min(8, mtiles - 8 * band), u = v - band * 8 * ntiles;
  const int m0 = (8 * band + u % bm) * T::BM, n0 = (u / bm) * RG;

  // A matrix' runs from byte `off` of the stage (or of the scales) of the workgroup's rows, which start with row tile t0 (a
  // group's first): where they lie and how far the next stage's do. Loads past the matrix read zeros.
  const KQ4MxDims dw = a.dw, dx = a.dx;
  auto runs = [](const uint8_t *m, const KQ4MxDims &d, int type, bool scales, int t0, int off, uint32_t &step) {
    const int tb = scales ? KQ4_MX_STILE : kq4_mx_tile_bytes(type), t = t0 + off / (8 * tb) * 8;
    const long all = (long)kq4_mx_size(d, type);
    long at = (scales ? (long)kq4_mx_codes_size(d, type) : 0) + kq4_mx_first(t, scales ? d.kq : d.kt) * tb + off % (8 * tb);
    if (t >= d.nt || at > all) at = all;
    step = t < d.nt ? (uint32_t)(kq4_mx_step(t, d.nt) * tb) : 0u;
    const long left = all - at;
    kq4_rsrc4 r = kq4_rsrc_at(m + at, (uint32_t)(left < 0x7fffffffL ? left : 0x7fffffffL), 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_readfirstlane(r[i]);   // (the wave's, in scalar registers)
    step = (uint32_t)__builtin_amdgcn_readfirstlane((int)step);
    return r;
  };
  uint32_t step_a, step_b, step_s[T::SPW];
  const kq4_rsrc4 ra = runs(a.x, dx, TYPE, false, m0 >> 4, wave * T::LA * 1024, step_a);
  constexpr int PER = T::B / G;                 // a stage's bytes of one weight matrix
  const int ob = wave * T::LB * 1024;
  const kq4_rsrc4 rb = runs(a.w[ob / PER], dw, 4, false, n0 >> 4, ob % PER, step_b);
  kq4_rsrc4 rs[T::SPW];
  constexpr int SA = T::BM / 16 * KQ4_MX_STILE, SB = T::BN / 16 / G * KQ4_MX_STILE;
#pragma unroll
  for (int l = 0; l < T::SPW; ++l) {
    const int o = (min(wave * T::SPW, T::SLOADS - T::SPW) + l) * 1024;
    if (o < SA) rs[l] = runs(a.x, dx, TYPE, true, m0 >> 4, o, step_s[l]);
    else rs[l] = runs(a.w[(o - SA) / SB], dw, 4, true, n0 >> 4, (o - SA) % SB, step_s[l]);
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t *)&lds[0];
  const uint32_t v16 = 16u * lane;
  const int nk = dw.kt, nq = dw.kq;
  auto load_stage = [&](int k, int slot) {      // (past the last stage: that one again, not used)
    const uint32_t kk = (uint32_t)min(k, nk - 1), to = lds0 + slot * T::STAGE;
    kq4_mx_load<T::LA>(ra, v16, kk * step_a, to + wave * T::LA * 1024);
    kq4_mx_load<T::LB>(rb, v16, kk * step_b, to + T::A + wave * T::LB * 1024);
  };
  auto load_scales = [&](int q) {
    const uint32_t qq = (uint32_t)min(q, nq - 1);
#pragma unroll
    for (int l = 0; l < T::SPW; ++l)
      kq4_mx_load<1>(rs[l], v16, qq * step_s[l],
                     lds0 + S * T::STAGE + (min(wave * T::SPW, T::SLOADS - T::SPW) + l) * 1024);
  };

  // the wave's tiles of 32 rows, as row tiles of 16 in the operand's part of LDS
  auto at = [&](int i) { return 2 * (TI * wm + i); };
  auto bt = [&](int j) { return G == 2 ? (j / (TJ / 2)) * (RG / 16) + TJ * wn + 2 * (j % (TJ / 2)) : 2 * (TJ * wn + j); };
  const int frag = l32 >> 4, r16 = l32 & 15;
  const uint8_t *la = lds + frag * T::TA, *lb = lds + T::A + frag * 1024, *ls = lds + S * T::STAGE + frag * KQ4_MX_STILE;

  kq4_v16f acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  kq4_v8i fa[2][TI], fb[2][TJ];
  uint32_t sa[2][TI], sb[2][TJ], na[2][TI], nb[2][TJ];
  auto read = [&](int s, int slot) {            // half s of the stage in a slot
    const int b = 2 * s + half, o = slot * T::STAGE;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const uint8_t *t = la + o + at(i) * T::TA;
      const uint4 x = *reinterpret_cast<const uint4 *>(t + kq4_mx_piece(b, r16));
      uint2 y = make_uint2(0u, 0u);
      if constexpr (TYPE == 6) y = *reinterpret_cast<const uint2 *>(t + kq4_mx_rest(b, r16));
      fa[s][i] = kq4_v8i{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const uint4 x = *reinterpret_cast<const uint4 *>(lb + o + bt(j) * 1024 + kq4_mx_piece(b, r16));
      fb[s][j] = kq4_v8i{(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0};
    }
  };
  auto read_scales = [&]() {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int o = (2 * s + half) * 64 + 4 * r16;
#pragma unroll
      for (int i = 0; i < TI; ++i) na[s][i] = *reinterpret_cast<const uint32_t *>(ls + at(i) * KQ4_MX_STILE + o);
#pragma unroll
      for (int j = 0; j < TJ; ++j)
        nb[s][j] = *reinterpret_cast<const uint32_t *>(ls + (T::BM / 16 + bt(j)) * KQ4_MX_STILE + o);
    }
  };
  auto take_scales = [&]() {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < TI; ++i) sa[s][i] = na[s][i];
#pragma unroll
      for (int j = 0; j < TJ; ++j) sb[s][j] = nb[s][j];
    }
  };
#define KQ4_MX_PRODUCTS(H, J)                                                                                     \
  _Pragma("unroll") for (int i = 0; i < TI; ++i) _Pragma("unroll") for (int j = 0; j < TJ; ++j) acc[i][j] =      \
      __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[H][i], fb[H][j], acc[i][j], kq4_mx_fmt<TYPE>, 4, J,      \
                                                      (int)sa[H][i], J, (int)sb[H][j]);
// products and LDS reads in turn: reads issued in a row hold the matrix unit up
#define KQ4_MX_INTERLEAVE                                                                                         \
  _Pragma("unroll") for (int z = 0; z < TI + TJ; ++z) {                                                           \
    __builtin_amdgcn_sched_group_barrier(0x8, TI * TJ / (TI + TJ), 0);                                            \
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                                            \
  }

  load_scales(0);
#pragma unroll
  for (int s = 0; s < S; ++s) load_stage(s, s);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * T::LPW) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  read_scales();
  take_scales();
  read(0, 0);
  int slot = 0;
  auto stage = [&](int k, auto jc) {
    constexpr int J = decltype(jc)::value;
    const int next = slot + 1 == S ? 0 : slot + 1;
    read(1, slot);
    KQ4_MX_PRODUCTS(0, J)
    KQ4_MX_INTERLEAVE
    __builtin_amdgcn_sched_barrier(0);
    // this wave's part of the next stage has come, and its reads of this one are done
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * T::LPW) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (J == 0) load_scales((k >> 2) + 1);
    load_stage(k + S, slot);
    read(0, next);
    if constexpr (J == 3) read_scales();
    KQ4_MX_PRODUCTS(1, J)
    KQ4_MX_INTERLEAVE
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (J == 3) take_scales();
    slot = next;
  };
  for (int k = 0; k < nk; k += 4) {
    stage(k, std::integral_constant<int, 0>{});
    if (k + 1 < nk) stage(k + 1, std::integral_constant<int, 1>{});
    if (k + 2 < nk) stage(k + 2, std::integral_constant<int, 2>{});
    if (k + 3 < nk) stage(k + 3, std::integral_constant<int, 3>{});
  }
#undef KQ4_MX_PRODUCTS
#undef KQ4_MX_INTERLEAVE
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the loads past the last stage: LDS is not given back before

  // The residual's loads of 32 tokens are all on their way before the first of them is waited for (it may be out: an
  // element is read and written by one lane). Past the edges they read the last row's or column's, which is not stored.
  const bool inside = m0 + T::BM <= a.n && n0 + RG <= a.rows;
  const int c0 = n0 + 32 * (TJ / G) * wn + l32;
#pragma unroll
  for (int i = 0; i < TI; ++i) {
    const int t0 = m0 + 32 * (TI * wm + i) + 4 * half;
    float y[16][TJ / G];
    if (a.res) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float *r = a.res + (size_t)min(t0 + 8 * (e >> 2) + (e & 3), a.n - 1) * a.ldo;
#pragma unroll
        for (int j = 0; j < TJ / G; ++j) y[e][j] = r[min(c0 + 32 * j, a.rows - 1)];
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int j = 0; j < TJ / G; ++j) {
        const float p = G == 2 ? kq4_mx_gate(acc[i][j][e], acc[i][G == 2 ? TJ / 2 + j : j][e]) : acc[i][j][e];
        y[e][j] = a.res ? p + y[e][j] : p;
      }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int tok = t0 + 8 * (e >> 2) + (e & 3);
      float *o = a.out + (size_t)tok * a.ldo + c0;
      if (inside) {
#pragma unroll
        for (int j = 0; j < TJ / G; ++j) o[32 * j] = y[e][j];
      } else if (tok < a.n) {
#pragma unroll
        for (int j = 0; j < TJ / G; ++j)
          if (c0 + 32 * j < a.rows) o[32 * j] = y[e][j];
      }
    }
  }
}

template <int TYPE, int G, int TI, int TJ, int WM, int WN, int S, int OCC>
static int launch(const KQ4MxArgs &a, hipStream_t s) {
  using T = KQ4MxTile<TYPE, TI, TJ, WM, WN, S>;
  auto *k = kq4_mx_gemm_kernel<TYPE, G, TI, TJ, WM, WN, S, OCC>;
  static std::atomic<unsigned long long> done{0};
  const hipError_t e = kq4_lds_limit_once(reinterpret_cast<const void *>(k), T::LDS, done);
  if (e != hipSuccess) return (int)e;
  const int mt = (a.n + T::BM - 1) / T::BM, nt = (a.rows + T::BN / G - 1) / (T::BN / G);
  hipLaunchKernelGGL(k, dim3((unsigned)mt * nt), dim3(64 * T::NW), T::LDS, s, a, mt, nt);
  return (int)hipGetLastError();
}

int kq4_launch_mx_gemm(const KQ4MxArgs &a, int type, hipStream_t s) {
  if (a.w[1]) return type == 4 ? launch<4, 2, 2, 4, 2, 2, 3, 2>(a, s) : launch<6, 2, 2, 4, 2, 2, 2, 2>(a, s);
  return type == 4 ? launch<4, 1, 2, 4, 2, 2, 3, 2>(a, s) : launch<6, 1, 2, 4, 2, 2, 2, 2>(a, s);
}
