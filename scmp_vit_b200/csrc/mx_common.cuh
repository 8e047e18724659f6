// Shared pieces of the microscaled 4-bit operators and the block operators
// around them (internal; the C ABI lives in include/scmp_b200.h).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/scmp_b200.h"

namespace scmp {

// ------------------------------------------------------------ element types

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

// Element i of an array of enum scmp_dtype.
__device__ __forceinline__ float load_as_f32(const void *p, int dtype, int64_t i) {
  if (dtype == SCMP_F32) return static_cast<const float *>(p)[i];
  if (dtype == SCMP_BF16) return to_f32(static_cast<const __nv_bfloat16 *>(p)[i]);
  return to_f32(static_cast<const __half *>(p)[i]);
}

// n / d for n < 2^32 by a multiplication and shifts (round-up method of Granlund
// and Montgomery: m = ceil(2^(32 + s) / d) - 2^32, s = ceil(log2 d)).
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t div) : d(div), m(0), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    const uint32_t t = __umulhi(n, m);
    return s ? (t + ((n - t) >> 1)) >> (s - 1) : n;
  }
};

// Two elements packed in a 32-bit word (16-bit types).
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// Elements of T in 16 bytes.
template <typename T> constexpr int kVec16 = 16 / (int)sizeof(T);

// 16 bytes of T <-> fp32 registers.
template <typename T> __device__ __forceinline__ void unpack16(const uint4 &u, float *v) {
  const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y), c = unpack2<T>(u.z), d = unpack2<T>(u.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}
template <> __device__ __forceinline__ void unpack16<float>(const uint4 &u, float *v) {
  v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y);
  v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
}
template <typename T> __device__ __forceinline__ uint4 pack16(const float *v) {
  return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                    pack2<T>(v[6], v[7]));
}
template <> __device__ __forceinline__ uint4 pack16<float>(const float *v) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                    __float_as_uint(v[3]));
}

// ------------------------------------------------------- 4-bit block formats

// Layout of a quantised [rows, K] operand.
//   data:   [rows][kp / 2] bytes, element 2i in the low nibble of byte i; kp = K
//           rounded up to 32, codes past K are 0, so every row starts 16-byte
//           aligned (what a tensor map asks of its strides).
//   scales: [ceil(rows / 128)][groups][512] bytes, groups = ceil(blocks / 4): the
//           atom of 128 rows x 4 block scales holds the scale of row r, block b
//           at (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4, which is the order the
//           tensor core's scale columns take from one 32-lane x 16-byte copy.
//           Scales of blocks past K and of rows past `rows` are 0 (a finite
//           value in both scale types).
struct MxLayout {
  int64_t rows, K, kp, groups;
  int block;  // elements per scale: 32 (e8m0) or 16 (e4m3)
  int64_t data_bytes() const { return rows * (kp / 2); }
  int64_t scale_bytes() const { return (rows + 127) / 128 * groups * 512; }
};
inline MxLayout mx_layout(int64_t rows, int64_t K, int fmt) {
  MxLayout l;
  l.rows = rows;
  l.K = K;
  l.block = fmt == SCMP_MXFP4 ? 32 : 16;
  l.kp = (K + 31) / 32 * 32;
  l.groups = (l.kp / l.block + 3) / 4;
  return l;
}
// Byte of the first scale of a group of four (row r, group g of `groups`).
__host__ __device__ inline int64_t mx_scale_word(int64_t r, int64_t g, int64_t groups) {
  return ((r >> 7) * groups + g) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// Eight fp32 values to eight e2m1 codes, value i in nibble i: round to nearest
// even, saturating at 6.
__device__ __forceinline__ uint32_t e2m1x8(const float *v) {
  uint32_t r;
  asm("{\n.reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n}\n"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Nearest e4m3 code of v >= 0, saturating at 448, and the value it stands for.
__device__ __forceinline__ uint32_t e4m3_code(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return (uint32_t)r & 0xFFu;
}
__device__ __forceinline__ float e4m3_value(uint32_t code) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)code));
  return __half2float(__ushort_as_half((unsigned short)(h2 & 0xFFFFu)));
}
// Value of an e8m0 code below 0xFF: 2^(code - 127); code 0 is subnormal in fp32.
__device__ __forceinline__ float e8m0_value(uint32_t code) {
  return __uint_as_float(code ? code << 23 : 0x00400000u);
}

constexpr uint32_t kMxNan = 0xFF;  // e8m0 NaN
constexpr uint32_t kNvNan = 0x7F;  // e4m3 NaN

// Magnitudes are compared as integers, the sign bit cleared: their order is the
// numbers' and every NaN lies above the infinities.
template <int N> __device__ __forceinline__ uint32_t max_bits(const float *v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

// One lane's eight consecutive values of a block whose largest magnitude has
// the bits `amax`: the block's scale code and the eight element codes.
//   mxfp4: scale 2^E, E = floor(log2 amax) - 2 (never below -127), read off
//   amax's exponent field; x * 2^-E is exact wherever it decides a code.
//   nvfp4: scale s = e4m3(amax * 2^-e * fl(1/6)), code of the correctly rounded
//   quotient x * 2^-e / s, from s's correctly rounded reciprocal with one
//   correction by the remainder (Markstein 1990).  s has 4 significant bits, so
//   a value on a border between two codes divides to exactly that border and
//   no other value rounds onto it: the codes are those of the exact quotient.
// A NaN or an infinity in the block: the NaN scale, element codes 0.
// kExp: nvfp4 with e != 0; x * 2^-e may then leave fp32's range, and is held to
// a magnitude that saturates under every scale.
template <int kFmt, bool kExp>
__device__ __forceinline__ uint32_t mx_encode8(const float *x, uint32_t amax, float inv_exp,
                                               uint32_t *codes) {
  const uint32_t field = amax >> 23;
  const bool bad = field == 0xFFu;
  float q[8];
  uint32_t scale;
  if (kFmt == SCMP_MXFP4) {
    scale = bad ? kMxNan : (field > 2 ? field - 2 : 0u);
    const float inv = __uint_as_float((254u - scale) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = x[i] * inv;
  } else {
    const float a = __uint_as_float(amax);
    scale = e4m3_code((kExp ? a * inv_exp : a) * (1.0f / 6.0f));
    const float s = e4m3_value(scale), r = scale ? __frcp_rn(s) : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = x[i];
      if (kExp) v = fminf(fmaxf(v * inv_exp, -1e30f), 1e30f);
      const float y = v * r;
      q[i] = copysignf(__fmaf_rn(__fmaf_rn(-y, s, v), r, y), v);  // -0 stays -0
    }
    if (bad) scale = kNvNan;
  }
  const uint32_t c = e2m1x8(q);
  *codes = bad ? 0u : c;
  return scale;
}

// --------------------------------------------------------------- launchers

cudaError_t launch_mx_quantize(const void *x, int dtype, int64_t ld, const MxLayout &l, int fmt,
                               int scale_exp, uint8_t *data, uint8_t *scales, cudaStream_t s);
cudaError_t launch_mx_dequantize(const uint8_t *data, const uint8_t *scales, const MxLayout &l,
                                 int fmt, int scale_exp, void *out, int dtype, cudaStream_t s);

struct MxProduct {
  const uint8_t *a, *a_scales, *b, *b_scales;
  int64_t M, N, K;
  int fmt;
  float alpha;  // 2^(a_exp + b_exp)
  const void *bias;  // nullable [N]
  int bias_dtype;
  void *out;  // [M, N] row-major
  int out_dtype;
};
// Activation rows per tile and tiles of 256 weight rows x that, over `pairs`.
struct MxTilePlan {
  int nt;
  uint32_t tiles_f, tiles;
};
MxTilePlan mx_tile_plan(int64_t M, int64_t N, int pairs);
cudaError_t launch_mx_matmul(const MxProduct &p, unsigned int *error, cudaStream_t s);
// A few rows: x quantised in the same launch, or NULL with p.a's codes.  Which
// products that launch can take, and where it is faster than quantise + tiles.
bool mx_thin_fits(int64_t M, int64_t K);
bool mx_thin(int64_t M, int64_t N, int64_t K);
cudaError_t launch_mx_thin(const MxProduct &p, const void *x, int x_dtype, int64_t ld,
                           cudaStream_t s);

}  // namespace scmp
