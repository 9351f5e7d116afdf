// kq4_mx_dev.h - device helpers of the microscaled kernels (gfx950).
#pragma once

#include "kq4_common.h"
#include "kq4_mx.h"

typedef float kq4_v4f __attribute__((ext_vector_type(4)));
typedef int kq4_v8i __attribute__((ext_vector_type(8)));
typedef float kq4_v16f __attribute__((ext_vector_type(16)));
typedef unsigned kq4_v6u __attribute__((ext_vector_type(6)));

// The 32 elements of a block with scale byte b, as the matrix unit holds them. The conversions divide by the scale and
// round to nearest, ties to even (subnormal scales and values included: measured over their boundaries); a block
// that is NaN gets codes 0.
template <int TYPE>
KQ4_DEV void kq4_mx_encode(const float (&v)[32], uint32_t b, uint32_t (&o)[TYPE]) {
  const float s = __uint_as_float(kq4_mx_scale_bits(b));
  if constexpr (TYPE == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[8 * i], v[8 * i + 1], s, 0);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[8 * i + 2], v[8 * i + 3], s, 1);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[8 * i + 4], v[8 * i + 5], s, 2);
      o[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[8 * i + 6], v[8 * i + 7], s, 3);
    }
  } else {   // (the instruction interleaves its operands)
    kq4_v16f even, odd;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      even[i] = v[2 * i];
      odd[i] = v[2 * i + 1];
    }
    const kq4_v6u u = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, s);
#pragma unroll
    for (int i = 0; i < 6; ++i) o[i] = u[i];
  }
#pragma unroll
  for (int i = 0; i < TYPE; ++i) o[i] = b == 255u ? 0u : o[i];
}

// A block's codes to and from its places in a tile.
template <int TYPE>
KQ4_DEV void kq4_mx_put(uint8_t *tile, int b, int r, const uint32_t (&o)[TYPE]) {
  *reinterpret_cast<uint4 *>(tile + kq4_mx_piece(b, r)) = make_uint4(o[0], o[1], o[2], o[3]);
  if constexpr (TYPE == 6) *reinterpret_cast<uint2 *>(tile + kq4_mx_rest(b, r)) = make_uint2(o[4], o[5]);
}
template <int TYPE>
KQ4_DEV void kq4_mx_get(const uint8_t *tile, int b, int r, uint32_t (&o)[TYPE]) {
  const uint4 v = *reinterpret_cast<const uint4 *>(tile + kq4_mx_piece(b, r));
  o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
  if constexpr (TYPE == 6) {
    const uint2 u = *reinterpret_cast<const uint2 *>(tile + kq4_mx_rest(b, r));
    o[4] = u.x; o[5] = u.y;
  }
}

// The matrix unit's name of a type.
template <int TYPE>
constexpr int kq4_mx_fmt = TYPE == 4 ? 4 : 2;

KQ4_DEV uint32_t kq4_absbits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// e^a as 2^(a log2 e) with that product's rounding put right to first order: off by at most 4 halves of an ulp (2 of the hardware's
// exp2, one each of the factor and the product with it).
KQ4_DEV float kq4_mx_exp(float a) {
  const float hi = a * 1.44269504f, lo = fmaf(a, 1.92596303e-8f, fmaf(a, 1.44269504f, -hi));
  return __builtin_amdgcn_exp2f(hi) * fmaf(lo, 0.693147181f, 1.0f);
}

// silu(g) = g / (1 + e^-g) for |g| <= 64. The quotient is the hardware's reciprocal (1 ulp) and one correction, so it is rounded once;
// with the sum's rounding that is 6 halves of an ulp of the result at most, 4 for g > 0.
KQ4_DEV float kq4_mx_silu(float g) {
  const float d = 1.0f + kq4_mx_exp(-g), r = __builtin_amdgcn_rcpf(d), q = g * r;
  return fmaf(fmaf(-q, d, g), r, q);
}

// silu(g) for any g. Above 64 it is g, and below -64 g e^(g/2) e^(g/2), as 1 + e^-g is 1 or e^-g there: nothing leaves the normal
// numbers before the result does (e^-g overflows below -88.7, where g e^g is normal down to -92). 10 halves of an ulp below -64, and
// half of the least subnormal. Past 200 in the exponent nothing of it is left.
KQ4_DEV float kq4_mx_silu_far(float g) {
  const float e = kq4_mx_exp(fmaxf(0.5f * g, -200.0f));
  return g > 64.0f ? g : g < -64.0f ? g * e * e : kq4_mx_silu(g);
}

// silu(g) * u of N gates of a lane, the same bits whichever way a wave goes. A wave asks once whether any gate is past 64, which
// few models have: 2048 x 6144 x 2048 40.3 us so, 45.2 with both forms of silu at every gate.
template <int N, class V>
KQ4_DEV V kq4_mx_gate(V g, V u) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(g[i]));
  if (__builtin_expect(__ballot(m > 64.0f) != 0, 0)) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = kq4_mx_silu_far(g[i]) * u[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = kq4_mx_silu(g[i]) * u[i];
  }
  return g;
}
