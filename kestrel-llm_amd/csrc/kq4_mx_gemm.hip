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
// 4096 x 4096 x 12288 without a residual: 97 us at 4 bits of the activations, 108 at 6, 4.2 and 3.8 PFLOP/s (the unit alone, fed
// from registers: 5.9 to 7.0). The matrix unit is busy half of the time at 1.83 to 1.87 of 2.4 GHz: the power that it takes
// lowers the clock, and 256 x 256 tiles, wave tiles of 128 x 128 and finer turns of loads and products came within 6 % of each
// other. Short K ends in its outputs: 2048 x 12288 x 4096 gated is 115 us, 94 without its 100 MB of stores, which the
// workgroups, all in step, send at once. Priorities that set a CU's two workgroups apart
// changed nothing. NT: outputs and residual go past the caches (launch_form has when).
template <int TYPE, int TI, int TJ, int WM, int WN, int S>
struct KQ4MxTile {
  static constexpr int NW = WM * WN, BM = 32 * TI * WM, BN = 32 * TJ * WN;
  static constexpr int TA = 256 * TYPE;                       // bytes of an activation tile (16 x 128)
  static constexpr int A = BM / 16 * TA, B = BN / 16 * 1024;  // a stage's operands
  static constexpr int STAGE = A + B;
  static constexpr int LA = (A / 1024 + NW - 1) / NW, LB = B / 1024 / NW, LPW = LA + LB;   // a wave's loads
  static constexpr int SCALES = (BM + BN) / 16 * KQ4_MX_STILE, SLOADS = SCALES / 1024;
  static constexpr int SPW = (SLOADS + NW - 1) / NW;
  static constexpr int LDS = S * STAGE + SCALES;
  // a wave's runs lie in one group of 8 row tiles, and (gated) in one matrix
  static_assert(B % (1024 * NW) == 0 && SLOADS % SPW == 0, "kq4_mx_gemm: runs per wave");
  // the first run of a wave's activations (where there are not as many for each, the last waves bring the last ones)
  static __device__ int first_a(int wave) { return wave * LA < A / 1024 - LA ? wave * LA : A / 1024 - LA; }
  static_assert(8 * TA % (LA * 1024) == 0 && 8 % LB == 0 && BM % 128 == 0 && BN % 128 == 0, "kq4_mx_gemm: groups");
  static_assert(LDS <= 160 * 1024, "kq4_mx_gemm: LDS");
};

// N runs of 1 KB from offset soff of r to LDS address `to` on: one address register for them all, the rest of it in the
// instructions' offset, which counts on both sides.
template <int N>
KQ4_DEV void kq4_mx_load(const kq4_rsrc4 &r, uint32_t v16, uint32_t soff, uint32_t to) {
  static_assert(N >= 1 && N <= 4, "kq4_mx_load: runs");
  if constexpr (N == 4)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds\n\t"
                 "buffer_load_dwordx4 %1, %2, %3 offen offset:1024 lds\n\tbuffer_load_dwordx4 %1, %2, %3 offen offset:2048 lds\n\t"
                 "buffer_load_dwordx4 %1, %2, %3 offen offset:%4 lds" ::"s"(to), "v"(v16), "s"(r), "s"(soff), "n"(3 * 1024)
                 : "memory", "m0");
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
}

template <int TYPE, int G, int TI, int TJ, int WM, int WN, int S, int OCC, bool NT>
__global__ __launch_bounds__(64 * WM * WN, OCC) void kq4_mx_gemm_kernel(KQ4MxArgs a, int mtiles, int ntiles, int ksplit, int per) {
  using T = KQ4MxTile<TYPE, TI, TJ, WM, WN, S>;
  constexpr int RG = T::BN / G;                 // output rows of the workgroup
  static_assert(RG % 128 == 0, "kq4_mx_gemm: whole groups of rows");
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM, l32 = lane & 31, half = lane >> 5;

  // XCD x works on a run of tiles, in bands of 8 tiles of tokens, so that what it reads at a time is shared
  const int all = mtiles * ntiles * ksplit, xcd = blockIdx.x & 7, q8 = all >> 3, r8 = all & 7;
  const int vs = xcd * q8 + (xcd < r8 ? xcd : r8) + (int)(blockIdx.x >> 3);
  const int slice = vs / (mtiles * ntiles), v = vs - slice * (mtiles * ntiles);
  const int band = v / (8 * ntiles), bm = min(8, mtiles - 8 * band), u = v - band * 8 * ntiles;
  const int m0 = (8 * band + u % bm) * T::BM, n0 = (u / bm) * RG;

  // Where a wave's runs lie (kq4_mx_run) as a buffer that ends with the matrix. Loads past it read zeros; what a run of the last
  // group holds past its row tiles belongs to rows that are not stored.
  const KQ4MxDims dw = kq4_mx_dims(a.rows, a.cols), dx = kq4_mx_dims(a.n, a.cols);
  const uint8_t *xq = static_cast<const uint8_t *>(a.x);
  auto runs = [](const uint8_t *m, const KQ4MxDims &d, int type, bool scales, int t0, int off, uint32_t &step) {
    const KQ4MxRun u = kq4_mx_run(d, type, scales, t0, off);
    kq4_rsrc4 r = kq4_rsrc_at(m + u.at, u.bytes, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_readfirstlane(r[i]);   // (the wave's, in scalar registers)
    step = (uint32_t)__builtin_amdgcn_readfirstlane((int)u.step);
    return r;
  };
  uint32_t step_a, step_b, step_s[T::SPW];
  const kq4_rsrc4 ra = runs(xq, dx, TYPE, false, m0 >> 4, T::first_a(wave) * 1024, step_a);
  constexpr int PER = T::B / G;                 // a stage's bytes of one weight matrix
  const int ob = wave * T::LB * 1024;
  const kq4_rsrc4 rb = runs(a.w[ob / PER], dw, 4, false, n0 >> 4, ob % PER, step_b);
  kq4_rsrc4 rs[T::SPW];
  constexpr int SA = T::BM / 16 * KQ4_MX_STILE, SB = T::BN / 16 / G * KQ4_MX_STILE;
#pragma unroll
  for (int l = 0; l < T::SPW; ++l) {
    const int o = (min(wave * T::SPW, T::SLOADS - T::SPW) + l) * 1024;
    if (o < SA) rs[l] = runs(xq, dx, TYPE, true, m0 >> 4, o, step_s[l]);
    else rs[l] = runs(a.w[(o - SA) / SB], dw, 4, true, n0 >> 4, (o - SA) % SB, step_s[l]);
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t *)&lds[0];
  const uint32_t v16 = 16u * lane;
  // the slice's stages and groups of four
  const int q0 = slice * per, nq = min(per, dw.kq - q0), nk = min(4 * per, dw.kt - 4 * q0);
  auto load_stage = [&](int k, int slot) {      // (past the last stage: that one again, not used)
    const uint32_t kk = (uint32_t)(4 * q0 + min(k, nk - 1)), to = lds0 + slot * T::STAGE;
    kq4_mx_load<T::LA>(ra, v16, kk * step_a, to + T::first_a(wave) * 1024);
    kq4_mx_load<T::LB>(rb, v16, kk * step_b, to + T::A + wave * T::LB * 1024);
  };
  auto load_scales = [&](int q) {
    const uint32_t qq = (uint32_t)(q0 + min(q, nq - 1));
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

  const int c0 = n0 + 32 * (TJ / G) * wn + l32;
  if (ksplit > 1) {   // the sums of a slice, [slice][matrix][token][row]
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int tok = m0 + 32 * (TI * wm + i) + 8 * (e >> 2) + 4 * half + (e & 3);
        float *o = a.part + ((size_t)slice * G * a.n + tok) * a.rows + c0;
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          const int c = 32 * (j % (TJ / G));
          if (tok < a.n && c0 + c < a.rows) o[(size_t)(j / (TJ / G)) * a.n * a.rows + c] = acc[i][j][e];
        }
      }
    return;
  }
  if constexpr (G == 2)
    if (a.q) {
      // The gated product as the activations of the next one: 32 tokens of each wave at a time go through LDS, where a thread
      // then finds a block of 32 columns. The workgroup's 128 columns are one column tile of the matrix.
      constexpr int LD = 128 + 4;
      static_assert(RG == 128 && 32 * WM * LD * 4 <= T::LDS, "kq4_mx_gemm: quantized outputs");
      float *buf = reinterpret_cast<float *>(lds);
      const KQ4MxDims dq = kq4_mx_dims(a.n, a.rows);
      const int kt = n0 >> 7;
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < TJ / 2; ++j) {
          const kq4_v16f h = kq4_mx_gate<16>(acc[i][j], acc[i][TJ / 2 + j]);
#pragma unroll
          for (int e = 0; e < 16; ++e) buf[(32 * wm + 8 * (e >> 2) + 4 * half + (e & 3)) * LD + 32 * (TJ / 2 * wn + j) + l32] = h[e];
        }
        __syncthreads();
        for (int u = threadIdx.x; u < 32 * WM * 4; u += 64 * T::NW) {
          const int row = u >> 2, b = u & 3, tok = m0 + 32 * (TI * (row >> 5) + i) + (row & 31);
          if (tok >= a.n) continue;
          float f[32];
          uint32_t m = 0, o[TYPE] = {}, sc = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 x = *reinterpret_cast<const float4 *>(&buf[row * LD + 32 * b + 4 * k]);
            f[4 * k] = x.x; f[4 * k + 1] = x.y; f[4 * k + 2] = x.z; f[4 * k + 3] = x.w;
          }
          if (n0 + 32 * b < a.rows) {
#pragma unroll
            for (int k = 0; k < 32; ++k) m = max(m, kq4_absbits(f[k]));
            sc = kq4_mx_scale_byte(m, TYPE);
            kq4_mx_encode<TYPE>(f, sc, o);
          }
          const int tile = tok >> 4;
          const long at = kq4_mx_first(tile, dq.kt) + (long)kt * kq4_mx_step(tile, dq.nt);
          kq4_mx_put<TYPE>(a.q + at * T::TA, b, tok & 15, o);
          uint8_t *ps = a.q + kq4_mx_codes_size(dq, TYPE) +
                        (kq4_mx_first(tile, dq.kq) + (long)(kt >> 2) * kq4_mx_step(tile, dq.nt)) * KQ4_MX_STILE;
          ps[kq4_mx_scale_at(4 * (kt & 3) + b, tok & 15)] = (uint8_t)sc;
          if (kt == dq.kt - 1)   // the column tiles that the scales' last tile has and the codes do not
            for (int k = (kt & 3) + 1; k < 4; ++k) ps[kq4_mx_scale_at(4 * k + b, tok & 15)] = 0;
        }
      }
      return;
    }
  // The residual's loads of 32 tokens are all on their way before the first of them is waited for (it may be out: an element
  // is read and written by one lane): 4096 x 4096 x 12288 with a residual 112 us, one element after the other 165. Past the
  // edges they read the last row's or column's, which is not stored.
  const bool inside = m0 + T::BM <= a.n && n0 + RG <= a.rows;
  auto store = [&](auto with_res) {
    constexpr bool RES = decltype(with_res)::value;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int t0 = m0 + 32 * (TI * wm + i) + 4 * half;
      float y[16][TJ / G];
      if constexpr (RES)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float *r = a.res + (size_t)min(t0 + 8 * (e >> 2) + (e & 3), a.n - 1) * a.ldo;
#pragma unroll
          for (int j = 0; j < TJ / G; ++j) {
            const float *p = r + min(c0 + 32 * j, a.rows - 1);
            y[e][j] = NT ? __builtin_nontemporal_load(p) : *p;
          }
        }
#pragma unroll
      for (int j = 0; j < TJ / G; ++j) {
        kq4_v16f p = acc[i][j];
        if constexpr (G == 2) p = kq4_mx_gate<16>(p, acc[i][TJ / 2 + j]);
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e][j] = RES ? p[e] + y[e][j] : p[e];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int tok = t0 + 8 * (e >> 2) + (e & 3);
        float *o = a.out + (size_t)tok * a.ldo + c0;
        if (inside) {
#pragma unroll
          for (int j = 0; j < TJ / G; ++j) {
            if constexpr (NT) __builtin_nontemporal_store(y[e][j], o + 32 * j);
            else o[32 * j] = y[e][j];
          }
        } else if (tok < a.n) {
#pragma unroll
          for (int j = 0; j < TJ / G; ++j)
            if (c0 + 32 * j < a.rows) o[32 * j] = y[e][j];
        }
      }
    }
  };
  if (a.res) store(std::true_type{});
  else store(std::false_type{});
}

// out = [res +] the slices' sums in slice order (gated: of both matrices). A thread four outputs of a token, 256 apart,
// with the loads of four slices on their way at a time.
template <int G>
__global__ __launch_bounds__(256) void kq4_mx_join_kernel(KQ4MxArgs a, int ksplit, int chunks) {
  const int t = (int)(blockIdx.x / (unsigned)chunks), c0 = ((int)blockIdx.x - t * chunks) * 1024 + (int)threadIdx.x;
  const size_t m = (size_t)a.n * a.rows;
  const float *p = a.part + (size_t)t * a.rows;
  float y[4][G] = {}, res[4];
  if (a.res)
#pragma unroll
    for (int i = 0; i < 4; ++i) res[i] = a.res[(size_t)t * a.ldo + min(c0 + 256 * i, a.rows - 1)];
  for (int s = 0; s < ksplit; s += 4) {
    float v[4][G][4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i][g][u] = p[((size_t)min(s + u, ksplit - 1) * G + g) * m + min(c0 + 256 * i, a.rows - 1)];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i][g] += s + u < ksplit ? v[i][g][u] : 0.0f;
  }
  kq4_v4f o = {y[0][0], y[1][0], y[2][0], y[3][0]};
  if constexpr (G == 2) o = kq4_mx_gate<4>(o, kq4_v4f{y[0][1], y[1][1], y[2][1], y[3][1]});
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c0 + 256 * i < a.rows) a.out[(size_t)t * a.ldo + c0 + 256 * i] = a.res ? o[i] + res[i] : o[i];
}

template <int TYPE, int G, int TI, int TJ, int WM, int WN, int S, int OCC, bool NT>
static int launch(const KQ4MxArgs &a, int ksplit, hipStream_t s) {
  using T = KQ4MxTile<TYPE, TI, TJ, WM, WN, S>;
  auto *k = kq4_mx_gemm_kernel<TYPE, G, TI, TJ, WM, WN, S, OCC, NT>;
  static std::atomic<unsigned long long> done{0};
  hipError_t e = kq4_lds_limit_once(reinterpret_cast<const void *>(k), T::LDS, done);
  if (e != hipSuccess) return (int)e;
  const int mt = (a.n + T::BM - 1) / T::BM, nt = (a.rows + T::BN / G - 1) / (T::BN / G);
  const int kq = kq4_mx_dims(a.rows, a.cols).kq, per = (kq + ksplit - 1) / ksplit;   // (every slice has some: kq4_mx_split)
  hipLaunchKernelGGL(k, dim3((unsigned)mt * nt * ksplit), dim3(64 * T::NW), T::LDS, s, a, mt, nt, ksplit, per);
  e = hipGetLastError();
  if (e != hipSuccess || ksplit == 1) return (int)e;
  const int chunks = (a.rows + 1023) / 1024;
  hipLaunchKernelGGL(kq4_mx_join_kernel<G>, dim3((unsigned)chunks * a.n), dim3(256), 0, s, a, ksplit, chunks);
  return (int)hipGetLastError();
}

// As many slices of whole groups as there are with `want` asked for.
int kq4_mx_split(int kq, int want) {
  if (want > kq) want = kq;
  if (want < 1) want = 1;
  const int per = (kq + want - 1) / want;
  return (kq + per - 1) / per;
}

// One matrix: tiles of 128 x 128 in 4 waves of 64 x 64, as long as three of them a CU hold the launch, since a stage of few
// workgroups is all latency and shorter for the smaller tile (512 x 4096 x 4096: 12.7 us, in 128 x 256 18.1; 2400 x 4096 x 4096
// 30.5 and 34.2; but 4096 x 4096 x 4096, two rounds, 44.0 and 38.6), with the deeper ring up to one and a half a CU (1322 x
// 2944 x 3744 15.0 against 15.5, but 1800 x 4096 x 4096 26.1 against 24.4). Two matrices, whose tiles of 128 x 128 would not be
// whole groups of rows: where workgroups are alone on their CUs they have 8 waves of 64 x 64 and a stage more, two waves per
// SIMD as elsewhere two workgroups have.
// Outputs and residuals of KQ4_MX_PAST_CACHE bytes and more go past the caches (non-temporal: 2048 x 12288 x 4096 of one
// matrix 69 -> 58 us, 4096 x 12288 x 1024 65 -> 44, with a residual 98 -> 85); the memory side's 256 MB hold smaller ones for
// what reads them next (1796 x 5127 x 64 with a residual 18 us, non-temporal 28; 2048 x 8192 x 512 17 and 20).
#define KQ4_MX_PAST_CACHE ((size_t)80 << 20)
template <int TYPE, int G>
static int launch_form(const KQ4MxArgs &a, int ksplit, int ncu, hipStream_t s) {
  const long tiles = (long)((a.n + 127) / 128) * ((a.rows + 127) / 128) * ksplit;
  if constexpr (G == 1) {
    if (2 * tiles <= 3L * ncu) return launch<TYPE, 1, 2, 2, 2, 2, TYPE == 4 ? 4 : 3, 2, false>(a, ksplit, s);
    if (tiles <= 3L * ncu) return launch<TYPE, 1, 2, 2, 2, 2, TYPE == 4 ? 3 : 2, 3, false>(a, ksplit, s);
  } else {
    if (tiles <= ncu) return launch<TYPE, 2, 2, 2, 2, 4, 3, 1, false>(a, ksplit, s);
  }
  const size_t bytes = ksplit > 1 || a.q ? 0 : (size_t)a.n * a.rows * (a.res ? 8 : 4);
  if (bytes >= KQ4_MX_PAST_CACHE) return launch<TYPE, G, 2, 4, 2, 2, TYPE == 4 ? 3 : 2, 2, true>(a, ksplit, s);
  return launch<TYPE, G, 2, 4, 2, 2, TYPE == 4 ? 3 : 2, 2, false>(a, ksplit, s);
}

int kq4_launch_mx_gemm(const KQ4MxArgs &a, int type, int ksplit, int ncu, hipStream_t s) {
  if (a.w[1]) return type == 4 ? launch_form<4, 2>(a, ksplit, ncu, s) : launch_form<6, 2>(a, ksplit, ncu, s);
  return type == 4 ? launch_form<4, 1>(a, ksplit, ncu, s) : launch_form<6, 1>(a, ksplit, ncu, s);
}

size_t kq4_mx_part_bytes(int n, int rows, int matrices, int ksplit) {
  return ksplit > 1 ? (size_t)ksplit * matrices * n * rows * sizeof(float) : 0;
}

// The form by estimated microseconds, fitted to the times of both forms and of 1 to 16 slices over 9 matrices and 24 to 1024
// tokens:
//   rows kernel   2.5 + 1.2 per million outputs + products at 0.7e9 a microsecond (6 bits 0.65e9; gated 0.85e9, 0.66e9)
//   GEMM          6.5 + its stages: of one matrix 0.21 (6 bits 0.265) for a tile a CU, 0.28 (0.32) a tile up to three; of
//                 two 0.38 (0.48) for a workgroup alone on its CU; 1.05 a round of two beyond
//   K in slices   2.5 for the second launch + the sums written and read at 4.5e6 bytes a microsecond
// e.g. 4096 x 4096, 6 bits: 256 tokens 9.4 us in the rows kernel against 13.7 (two slices) and 13.2 in the GEMM, 768 20.5 against
// 21.7 and 14.7; 4096 x 12288, 512 tokens: 30.0 in two slices, 39.9 in one, 45.4 in the rows kernel. Over 556 launches its choices
// take 1.005 times the best ones (geometric mean), 1.31 times at most: gated pairs of 65 to 127 tokens past a tile a CU, whose second
// tile of 64 tokens the rows kernel works on whole, where the estimate counts tokens (100 x 12288 x 4096, 6 bits: estimated 19.2 us,
// 29.9, in two slices of the GEMM 22.9).
KQ4MxPlan kq4_mx_plan(int n, int rows, int cols, int matrices, int type, int ncu, int force_form, int force_split) {
  const KQ4MxDims d = kq4_mx_dims(rows, cols);
  const double outputs = (double)n * rows, products = outputs * cols * matrices;
  const double rate = matrices == 2 ? (type == 4 ? 0.85e9 : 0.66e9) : (type == 4 ? 0.7e9 : 0.65e9);
  KQ4MxPlan best = {0, 1};
  double least = 2.5 + 1.2e-6 * outputs + products / rate;
  const double tiles = (double)((n + 127) / 128) * ((rows + 127) / 128);
  // what is forced is done where its launches have fewer than 2^32 threads
  if (n <= 16 || (force_form == 1 && (double)d.nt * ((n + 15) >> 4) < 1 << 23)) least = 0.0;   // (a token tile: no GEMM)
  if (force_form == 2) least = 1e30;
  force_split = min(force_split, d.kq);
  if (tiles * force_split >= 1 << 23 || (double)((rows + 1023) / 1024) * n >= 1 << 24) force_split = 1;
  for (int want = 1; want <= 16; want *= 2) {
    if (force_split > 0 && want > 1) break;
    const int ks = kq4_mx_split(d.kq, force_split > 0 ? force_split : want);
    const double wgs = tiles * ks;
    if (want > 1 && (ks <= best.ksplit || wgs > (matrices == 1 ? 3.0 : 2.0) * ncu || kq4_mx_part_bytes(n, rows, matrices, ks) > KQ4_MX_PART_MAX)) break;
    const int stages = 4 * ((d.kq + ks - 1) / ks);
    const double wide = matrices == 1 ? (double)((n + 127) / 128) * ((rows + 255) / 256) * ks : wgs;
    double us = 1.05 * (double)(long)((wide + 2 * ncu - 1) / (2 * ncu));
    if (matrices == 2 && wgs <= ncu) us = type == 4 ? 0.38 : 0.48;
    if (matrices == 1 && wgs <= 3.0 * ncu) us = wgs <= ncu ? (type == 4 ? 0.21 : 0.265) : (type == 4 ? 0.28 : 0.32) * (wgs / ncu);
    us = 6.5 + stages * us;
    if (ks > 1) us += 2.5 + (ks + 1.5) * matrices * outputs * 4.0 / 4.5e6;
    if (us < least) {
      least = us;
      best = {1, ks};
    }
  }
  return best;
}
