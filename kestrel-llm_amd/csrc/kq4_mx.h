// kq4_mx.h - microscaled matrices: where an element and a scale lie (include/kq4.h has the layout in words). Plain
// integer arithmetic without device code, so host programs compile it too.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "kq4_kv.h"   // KQ4_HD

#define KQ4_MX_GROUP 8         // row tiles of 16 that lie side by side for each 128 columns
#define KQ4_MX_STILE 256       // bytes of a scale tile: 16 rows x 512 columns

// Bytes of a code tile: 16 rows x 128 columns of `type` (4 or 6) bits.
KQ4_HD int kq4_mx_tile_bytes(int type) { return 256 * type; }

// Row tiles, column tiles of codes (128) and of scales (512).
struct KQ4MxDims {
  int nt, kt, kq;
};
KQ4_HD KQ4MxDims kq4_mx_dims(int rows, int cols) {
  KQ4MxDims d;
  d.nt = (rows + 15) >> 4;
  d.kt = (cols + 127) >> 7;
  d.kq = (cols + 511) >> 9;
  return d;
}

// Tile k of row tile t is number kq4_mx_first(t) + k * kq4_mx_step(t): a group's row tiles lie side by side, so the
// tiles that a workgroup of 128 rows reads next are 8 consecutive ones.
KQ4_HD int kq4_mx_step(int t, int nt) {
  const int left = nt - (t & ~(KQ4_MX_GROUP - 1));
  return left < KQ4_MX_GROUP ? left : KQ4_MX_GROUP;
}
KQ4_HD long kq4_mx_first(int t, int kt) {
  return (long)(t & ~(KQ4_MX_GROUP - 1)) * kt + (t & (KQ4_MX_GROUP - 1));
}

KQ4_HD size_t kq4_mx_codes_size(const KQ4MxDims &d, int type) {
  return (size_t)d.nt * d.kt * kq4_mx_tile_bytes(type);
}
KQ4_HD size_t kq4_mx_size(const KQ4MxDims &d, int type) {
  return kq4_mx_codes_size(d, type) + (size_t)d.nt * d.kq * KQ4_MX_STILE;
}

// Runs of 1 KB that the GEMM loads a stage at a time: byte `off` of the code tiles (or the scale tiles) of a column tile's row
// tiles t0, t0 + 1, ... (t0 a group's first). `at`: where the first stage's lies; `step`: how far on the next stage's is;
// `bytes`: what the matrix holds from `at` on. A run that starts past the last row tile has no bytes and no step. The range
// check takes the scalar offset (stages times `step`) from `bytes` before it compares, unsigned: of a run that starts in the
// matrix every stage's start is in it too, so nothing is taken from less.
struct KQ4MxRun {
  long at;
  uint32_t bytes, step;
};
KQ4_HD KQ4MxRun kq4_mx_run(const KQ4MxDims &d, int type, bool scales, int t0, int off) {
  const int tb = scales ? KQ4_MX_STILE : kq4_mx_tile_bytes(type), t = t0 + off / (8 * tb) * 8, in = off % (8 * tb);
  const long all = (long)kq4_mx_size(d, type);
  KQ4MxRun r = {all, 0u, 0u};
  if (t + in / tb >= d.nt) return r;
  r.at = (scales ? (long)kq4_mx_codes_size(d, type) : 0) + kq4_mx_first(t, scales ? d.kq : d.kt) * tb + in;
  r.step = (uint32_t)(kq4_mx_step(t, d.nt) * tb);
  r.bytes = (uint32_t)(all - r.at < 0x7fffffffL ? all - r.at : 0x7fffffffL);
  return r;
}

// In a code tile: the first 16 bytes of row r's block b of 4, and the last 8 of its 24 (6 bits).
KQ4_HD int kq4_mx_piece(int b, int r) { return 256 * b + 16 * r; }
KQ4_HD int kq4_mx_rest(int b, int r) { return 1024 + 128 * b + 8 * r; }
// In a scale tile: the byte of row r and block b of the tile's 16.
KQ4_HD int kq4_mx_scale_at(int b, int r) { return 64 * (b & 3) + 4 * r + (b >> 2); }

// The scale byte of a block whose largest magnitude has the bits `amax` (sign clear): the exponent e + 127 of the
// least e >= -127 for which amax / 2^e, rounded to the element's precision, is not above the largest element. For
// e2m1 amax = 1.75 * 2^k and up rounds to 2^(k + 1) (7 is a tie between 6 and 8 and goes to 8, whose code is even),
// for e2m3 1.9375 * 2^k and up (7.75, between 7.5 and 8): the sum carries into the exponent just there. 255 where the
// block holds a NaN or infinity.
KQ4_HD uint32_t kq4_mx_scale_byte(uint32_t amax, int type) {
  if (amax >= 0x7f800000u) return 255u;
  const int b = (int)((amax + (type == 4 ? 0x200000u : 0x80000u)) >> 23) - 2;
  return b < 0 ? 0u : (uint32_t)b;
}
// 2^(b - 127) as fp32 bits (b = 0: a subnormal; 255, NaN, is not asked for).
KQ4_HD uint32_t kq4_mx_scale_bits(uint32_t b) { return b ? b << 23 : 0x400000u; }
