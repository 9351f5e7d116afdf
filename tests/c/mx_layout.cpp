// kq4_mx.h for a host program, through C entries (test_mx_layout.py).
#include "../../kestrel-llm_amd/csrc/kq4_mx.h"

extern "C" {
void t_dims(int rows, int cols, int *o) {
  const KQ4MxDims d = kq4_mx_dims(rows, cols);
  o[0] = d.nt;
  o[1] = d.kt;
  o[2] = d.kq;
}
size_t t_size(int rows, int cols, int type) { return kq4_mx_size(kq4_mx_dims(rows, cols), type); }
size_t t_codes(int rows, int cols, int type) { return kq4_mx_codes_size(kq4_mx_dims(rows, cols), type); }
// offset of byte y of the block that starts with column c of row r, and of its scale byte
long t_code_at(int rows, int cols, int type, int r, int c, int y) {
  const KQ4MxDims d = kq4_mx_dims(rows, cols);
  const int t = r >> 4, k = c >> 7, b = (c & 127) >> 5;
  return (kq4_mx_first(t, d.kt) + (long)k * kq4_mx_step(t, d.nt)) * kq4_mx_tile_bytes(type) +
         (y < 16 ? kq4_mx_piece(b, r & 15) + y : kq4_mx_rest(b, r & 15) + y - 16);
}
long t_scale_at(int rows, int cols, int type, int r, int c) {
  const KQ4MxDims d = kq4_mx_dims(rows, cols);
  const int t = r >> 4, q = c >> 9;
  return (long)kq4_mx_codes_size(d, type) + (kq4_mx_first(t, d.kq) + (long)q * kq4_mx_step(t, d.nt)) * KQ4_MX_STILE +
         kq4_mx_scale_at((c >> 5) & 15, r & 15);
}
unsigned t_scale_byte(unsigned amax, int type) { return kq4_mx_scale_byte(amax, type); }
unsigned t_scale_bits(unsigned b) { return kq4_mx_scale_bits(b); }
}
