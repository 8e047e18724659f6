// Shared pieces of the 8-bit operators: e4m3 codes with one power-of-two scale
// per block of 128 (internal; the C ABI lives in include/scmp_b200.h).
#pragma once

#include "mx_common.cuh"

namespace scmp {

constexpr int kFp8Block = 128;

// Layout of a quantised [rows, K] operand.
//   data:   [rows][kp] bytes, kp = K rounded up to 128, so that a tensor map sees
//           rows of whole blocks; codes past K are 0.
//   scales: [ceil(rows / 128)][groups][512] bytes, groups = ceil(ceil(K / 128) / 4),
//           the scale of row r, block b in the order of the 4-bit formats' atoms
//           (mx_scale_word): e8m0, 2^(code - 127).  A 128 x 128 block's scale
//           stands once in each of its rows, so that products read one layout.
//           Scales of blocks past K and of rows past `rows` are 0.
struct Fp8Layout {
  int64_t rows, K, kp, blocks, groups;
  int64_t data_bytes() const { return rows * kp; }
  int64_t scale_bytes() const { return (rows + 127) / 128 * groups * 512; }
};
inline Fp8Layout fp8_layout(int64_t rows, int64_t K) {
  Fp8Layout l;
  l.rows = rows;
  l.K = K;
  l.blocks = (K + kFp8Block - 1) / kFp8Block;
  l.kp = l.blocks * kFp8Block;
  l.groups = (l.blocks + 3) / 4;
  return l;
}
__host__ __device__ inline int64_t fp8_scale_at(int64_t r, int64_t b, int64_t groups) {
  return mx_scale_word(r, b >> 2, groups) + (b & 3);
}

constexpr uint32_t kFp8Nan = 0xFF;  // e8m0 NaN: a block that holds a NaN or an infinity

// Scale code of a block whose largest magnitude has the bits `amax`: the
// smallest power of two, from 2^-127 on, under which the block stays within
// e4m3's 448 = 1.75 2^8.  Powers of two cost the codes no accuracy (they are
// floating point), at most one of e4m3's 18 binades, and let the tensor core
// apply them.
__device__ __forceinline__ uint32_t fp8_scale(uint32_t amax) {
  // a significand above 1.75 (0x600000) carries into the exponent field of E + 8
  const uint32_t e = (amax + 0x1FFFFFu) >> 23;
  return amax >= 0x7F800000u ? kFp8Nan : max(e, 8u) - 8u;
}
// What values are multiplied by before they are rounded: 2^-E, and NaN blocks by
// 0 (their codes do not matter).  2^127 is a normal number, and code 0's; the
// largest code, 247, gives 2^-120.
__device__ __forceinline__ float fp8_inverse(uint32_t scale) {
  return __uint_as_float(scale == kFp8Nan ? 0u : (254u - scale) << 23);
}
__device__ __forceinline__ float fp8_value_of_scale(uint32_t scale) {
  return scale == kFp8Nan ? __uint_as_float(0x7FC00000u) : e8m0_value(scale);
}

// Two values to two e4m3 codes, `lo` in the low byte: to nearest even, saturating
// (a NaN block's 0 * infinity becomes the NaN code, which its scale makes one too).
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | e4m3x2(c, d) << 16;
}
// Four codes to their values.
__device__ __forceinline__ void e4m3_values(uint32_t codes, float *v) {
  uint32_t lo, hi;
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\n"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
  const float2 a = unpack2<__half>(lo), b = unpack2<__half>(hi);
  v[0] = a.x;
  v[1] = a.y;
  v[2] = b.x;
  v[3] = b.y;
}

// --------------------------------------------------------------- launchers

// x [rows, K] of `dtype`, rows `ld` apart.  Blocks: 1 x 128 (square false) or 128
// x 128.  data / scales: x's codes, nullable; t_data / t_scales: the codes of its
// transpose [K, rows] (of blocks of 128 rows x 1, or the same squares), nullable.
// column_sums: nullable [ceil(rows / 128)][K] fp32, sums over the rows of a block.
struct Fp8Quantize {
  const void *x;
  int dtype;
  int64_t rows, K, ld;
  bool square;
  uint8_t *data, *scales, *t_data, *t_scales;
  float *column_sums;
};
cudaError_t launch_fp8_quantize(const Fp8Quantize &q, cudaStream_t s);
cudaError_t launch_fp8_dequantize(const uint8_t *data, const uint8_t *scales, const Fp8Layout &l,
                                  void *out, int dtype, cudaStream_t s);
// out [K] = the column sums' sum over `parts` blocks, in their order.
cudaError_t launch_fp8_sum_columns(const float *sums, int64_t parts, int64_t K, void *out,
                                   int dtype, cudaStream_t s);

struct Fp8Product {
  const uint8_t *a, *a_scales, *b, *b_scales;
  int64_t M, N, K;
  const void *bias;  // nullable [N]
  int bias_dtype;
  void *out;  // [M, N] row-major
  int out_dtype;
};
// Rows of a per tile: w[0] throughout, or w[0] and w[1] in turn.  A unit is 256
// rows of b by the widths' sum.
struct Fp8TilePlan {
  int w[2];
  uint32_t tiles_f, units;  // tiles of 256 rows of b; units, those fastest
};
Fp8TilePlan fp8_tile_plan(int64_t M, int64_t N, int64_t K, int pairs);
// (counts its launches)
cudaError_t launch_fp8_matmul(const Fp8Product &p, unsigned int *error, cudaStream_t s);
// A few rows: x quantised in the same launch, or NULL with p.a's codes.
bool fp8_thin_fits(int64_t M, int64_t K);
bool fp8_thin(int64_t M, int64_t N, int64_t K);
cudaError_t launch_fp8_thin(const Fp8Product &p, const void *x, int x_dtype, int64_t ld,
                            cudaStream_t s);

}  // namespace scmp
