// kq4_mx.hip - microscaled matrices: fp32 rows quantized into one, and the way between a checkpoint's row-major codes
// and scales and the products' tiles.
#include "kq4_internal.h"
#include "kq4_mx_dev.h"

// Quantisation. A workgroup takes 16 rows x 512 columns (a scale tile), a thread one block of 32. The rows come in
// by 16-byte loads of consecutive lanes and go through LDS (rows 16 bytes apart in the banks, so that the eight lanes
// that read together hit different ones); a wave then writes one code tile, 1 or 1.5 KB in one run, and the scale
// bytes are gathered in LDS for one 256-byte run. Bound by memory: 4 bytes read, 17/32 or 25/32 written per element;
// 4096 x 12288 to 4 bits 38.5 us, 5.9 TB/s. All eight loads are on their way before the first is used, without branches
// (edges read the last row or columns again) and non-temporal: 46.9 us with a branch at each; a thread that loads its own
// block directly, 128 bytes from its neighbour's, took 59.
#define KQ4_MXQ_LD (512 + 4)
template <int TYPE>
__global__ __launch_bounds__(256) void kq4_mx_quantize_kernel(uint8_t *__restrict__ m, const float *__restrict__ x,
                                                              long ldx, int rows, int cols, KQ4MxDims d) {
  __shared__ __align__(16) float tile[16 * KQ4_MXQ_LD];
  __shared__ __align__(4) uint8_t sc[256];
  const int q = blockIdx.x % d.kq, t = blockIdx.x / d.kq;
  const int tid = threadIdx.x, c0 = 512 * q;
  uint4 ld[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 2 * i + (tid >> 7), c = 4 * (tid & 127);
    ld[i] = kq4_ld_nt(x + (size_t)min(16 * t + r, rows - 1) * ldx + min(c0 + c, cols - 4));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 2 * i + (tid >> 7), c = 4 * (tid & 127);
    const bool in = 16 * t + r < rows && c0 + c < cols;
    *reinterpret_cast<uint4 *>(&tile[r * KQ4_MXQ_LD + c]) = in ? ld[i] : make_uint4(0u, 0u, 0u, 0u);
  }
  __syncthreads();
  const int r = tid & 15, b = tid >> 4;
  float v[32];
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 f = *reinterpret_cast<const float4 *>(&tile[r * KQ4_MXQ_LD + 32 * b + 4 * i]);
    v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) a = max(a, kq4_absbits(v[i]));
  const uint32_t s = kq4_mx_scale_byte(a, TYPE);
  uint32_t o[TYPE];
  kq4_mx_encode<TYPE>(v, s, o);
  const int k = 4 * q + (b >> 2);
  if (k < d.kt) {
    uint8_t *p = m + (kq4_mx_first(t, d.kt) + (long)k * kq4_mx_step(t, d.nt)) * (256 * TYPE);
    kq4_mx_put<TYPE>(p, b & 3, r, o);
  }
  sc[kq4_mx_scale_at(b, r)] = (uint8_t)s;
  __syncthreads();
  if (tid < 64) {
    uint8_t *p = m + kq4_mx_codes_size(d, TYPE) + (kq4_mx_first(t, d.kq) + (long)q * kq4_mx_step(t, d.nt)) * KQ4_MX_STILE;
    reinterpret_cast<uint32_t *>(p)[tid] = reinterpret_cast<const uint32_t *>(sc)[tid];
  }
}

// Between row-major codes [rows][cols * TYPE / 8] with scales [rows][cols / 32] and the tiles; a thread a block of a
// row, 16 rows x 16 blocks a workgroup. Packing fills what lies past the rows and columns with zeros.
template <int TYPE, bool PACK>
__global__ __launch_bounds__(256) void kq4_mx_pack_kernel(uint8_t *m, uint8_t *codes, uint8_t *scales, int rows,
                                                          int cols, KQ4MxDims d) {
  const int q = blockIdx.x % d.kq, t = blockIdx.x / d.kq;
  const int r = threadIdx.x & 15, b = threadIdx.x >> 4, row = 16 * t + r, blk = 16 * q + b, k = 4 * q + (b >> 2);
  const bool in = row < rows && 32 * blk < cols;
  uint8_t *p = m + (kq4_mx_first(t, d.kt) + (long)k * kq4_mx_step(t, d.nt)) * (256 * TYPE);
  uint8_t *ps = m + kq4_mx_codes_size(d, TYPE) +
                (kq4_mx_first(t, d.kq) + (long)q * kq4_mx_step(t, d.nt)) * KQ4_MX_STILE + kq4_mx_scale_at(b, r);
  const size_t at = (size_t)row * (cols / 32) + blk;
  uint2 *c = reinterpret_cast<uint2 *>(codes + at * (4 * TYPE));   // (24-byte blocks are 8-byte aligned)
  uint32_t o[TYPE] = {};
  if constexpr (PACK) {
    if (in)
#pragma unroll
      for (int i = 0; i < TYPE / 2; ++i) {
        const uint2 v = c[i];
        o[2 * i] = v.x;
        o[2 * i + 1] = v.y;
      }
    if (k < d.kt) kq4_mx_put<TYPE>(p, b & 3, r, o);
    *ps = in ? scales[at] : (uint8_t)0;
  } else if (in) {
    kq4_mx_get<TYPE>(p, b & 3, r, o);
#pragma unroll
    for (int i = 0; i < TYPE / 2; ++i) c[i] = make_uint2(o[2 * i], o[2 * i + 1]);
    scales[at] = *ps;
  }
}

int kq4_launch_mx_quantize(uint8_t *m, const float *x, long ldx, int rows, int cols, int type, hipStream_t s) {
  const KQ4MxDims d = kq4_mx_dims(rows, cols);
  const dim3 grid((unsigned)d.nt * d.kq);
  if (type == 4)
    hipLaunchKernelGGL((kq4_mx_quantize_kernel<4>), grid, dim3(256), 0, s, m, x, ldx, rows, cols, d);
  else
    hipLaunchKernelGGL((kq4_mx_quantize_kernel<6>), grid, dim3(256), 0, s, m, x, ldx, rows, cols, d);
  return (int)hipGetLastError();
}

int kq4_launch_mx_pack(uint8_t *m, uint8_t *codes, uint8_t *scales, int rows, int cols, int type, bool pack,
                       hipStream_t s) {
  const KQ4MxDims d = kq4_mx_dims(rows, cols);
  const dim3 grid((unsigned)d.nt * d.kq);
  auto *k = type == 4 ? (pack ? kq4_mx_pack_kernel<4, true> : kq4_mx_pack_kernel<4, false>)
                      : (pack ? kq4_mx_pack_kernel<6, true> : kq4_mx_pack_kernel<6, false>);
  hipLaunchKernelGGL(k, grid, dim3(256), 0, s, m, codes, scales, rows, cols, d);
  return (int)hipGetLastError();
}
