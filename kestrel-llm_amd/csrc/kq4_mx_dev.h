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

// silu(g) * u = g / (1 + e^-g) * u, e^-g as 2^(-g log2 e) with the product's rounding put right to first order: off by less
// than 2^-21 of the result (1 ulp each of exp2 and the reciprocal, half of one each of four others). exp may overflow: g / inf
// is the limit, and past 200 nothing of it is left either way.
KQ4_DEV float kq4_mx_gate(float g, float u) {
  const float a = -__builtin_amdgcn_fmed3f(g, -200.0f, 200.0f), hi = a * 1.44269504f;
  const float lo = fmaf(a, 1.92596303e-8f, fmaf(a, 1.44269504f, -hi));
  const float e = __builtin_amdgcn_exp2f(hi) * fmaf(lo, 0.693147181f, 1.0f);
  return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}
