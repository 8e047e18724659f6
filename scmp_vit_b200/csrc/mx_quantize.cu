// Quantisation to microscaled 4-bit floating point and back.
#include "mx_common.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;

// Eight consecutive elements of a row at column k (those at or past K are 0).
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T *__restrict__ row, int64_t k, int64_t K, float *v) {
  if (kVec && k + 8 <= K) {
    const uint4 *p = reinterpret_cast<const uint4 *>(row + k);
    if (sizeof(T) == 4) {
      unpack16<T>(__ldg(p), v);
      unpack16<T>(__ldg(p + 1), v + 4);
    } else {
      unpack16<T>(__ldg(p), v);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f32(row[k + i]) : 0.0f;
}

// One warp per 256 columns of one row: a lane holds eight consecutive values,
// the block's largest magnitude is a maximum over 4 (mxfp4) or 2 (nvfp4)
// lanes, every lane stores 4 bytes of codes and each fourth block's first lane
// one word of four scales.
template <typename T, int kFmt, bool kVec>
__global__ void __launch_bounds__(kThreads)
    mx_quantize_kernel(const T *__restrict__ x, int64_t ld, int64_t rows, int64_t K, int64_t kp,
                       int64_t groups, float inv_exp, uint8_t *__restrict__ data,
                       uint8_t *__restrict__ scales) {
  constexpr int kLanes = kFmt == SCMP_MXFP4 ? 4 : 2;  // lanes per block
  const int lane = threadIdx.x & 31;
  const int64_t chunks = (kp + 255) >> 8;
  const int64_t padded = (rows + 127) / 128 * 128;  // rows whose scales exist
  const int64_t units = padded * chunks;
  for (int64_t u = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5; u < units;
       u += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t r = u / chunks, k = (u % chunks) * 256 + lane * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (r < rows && k < K) load8<T, kVec>(x + r * ld, k, K, v);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max_nan(amax, fabsf(v[i]));
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) amax = max_nan(amax, __shfl_xor_sync(~0u, amax, o));
    uint32_t codes;
    const uint32_t scale = mx_encode8<kFmt>(v, amax, inv_exp, &codes);
    if (r < rows && k < kp) *reinterpret_cast<uint32_t *>(data + r * (kp >> 1) + (k >> 1)) = codes;
    uint32_t word = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      word |= __shfl_sync(~0u, scale, (lane & ~(4 * kLanes - 1)) + b * kLanes) << (8 * b);
    const int64_t g = k / (32 * kLanes);  // 8 values x kLanes lanes x 4 blocks
    if ((lane & (4 * kLanes - 1)) == 0 && g < groups)
      *reinterpret_cast<uint32_t *>(scales + mx_scale_word(r, g, groups)) = word;
  }
}

// Eight consecutive elements per thread.
template <typename T, int kFmt>
__global__ void __launch_bounds__(kThreads)
    mx_dequantize_kernel(const uint8_t *__restrict__ data, const uint8_t *__restrict__ scales,
                         int64_t rows, int64_t K, int64_t kp, int64_t groups, float exp_value,
                         T *__restrict__ out) {
  constexpr int kBlock = kFmt == SCMP_MXFP4 ? 32 : 16;
  const int64_t per = kp >> 3;
  const bool vec = (K & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  for (int64_t u = (int64_t)blockIdx.x * kThreads + threadIdx.x; u < rows * per;
       u += (int64_t)gridDim.x * kThreads) {
    const int64_t r = u / per, k = (u % per) * 8;
    const uint32_t codes =
        __ldg(reinterpret_cast<const uint32_t *>(data + r * (kp >> 1) + (k >> 1)));
    const int64_t b = k / kBlock;
    const uint32_t sc = __ldg(scales + mx_scale_word(r, b >> 2, groups) + (b & 3));
    float s;
    if (kFmt == SCMP_MXFP4)
      s = sc == kMxNan ? __uint_as_float(0x7FC00000u) : e8m0_value(sc);
    else
      s = e4m3_value(sc) * exp_value;
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t h2;
      asm("{\n.reg .b8 b, z1, z2, z3;\nmov.b32 {b, z1, z2, z3}, %1;\n"
          "cvt.rn.f16x2.e2m1x2 %0, b;\n}\n"
          : "=r"(h2)
          : "r"(codes >> (8 * i)));
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h2));
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
    T *dst = out + r * K + k;
    if (vec && k + 8 <= K) {
      uint4 *p = reinterpret_cast<uint4 *>(dst);
      p[0] = pack16<T>(v);
      if (sizeof(T) == 4) p[1] = pack16<T>(v + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < K) dst[i] = from_f32<T>(v[i]);
    }
  }
}

unsigned grid_for(int64_t threads) {
  const int64_t b = (threads + kThreads - 1) / kThreads;
  return (unsigned)(b < 148 * 8 ? b : 148 * 8);
}

template <typename T, int kFmt>
cudaError_t quantize(const void *x, int64_t ld, const MxLayout &l, int scale_exp, uint8_t *data,
                     uint8_t *scales, cudaStream_t s) {
  const float inv_exp = ldexpf(1.0f, -scale_exp);
  const int64_t warps = (l.rows + 127) / 128 * 128 * ((l.kp + 255) / 256);
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
  if (vec)
    mx_quantize_kernel<T, kFmt, true><<<grid_for(warps * 32), kThreads, 0, s>>>(
        static_cast<const T *>(x), ld, l.rows, l.K, l.kp, l.groups, inv_exp, data, scales);
  else
    mx_quantize_kernel<T, kFmt, false><<<grid_for(warps * 32), kThreads, 0, s>>>(
        static_cast<const T *>(x), ld, l.rows, l.K, l.kp, l.groups, inv_exp, data, scales);
  return cudaGetLastError();
}

template <typename T>
cudaError_t dequantize(const uint8_t *data, const uint8_t *scales, const MxLayout &l, int fmt,
                       int scale_exp, void *out, cudaStream_t s) {
  const unsigned grid = grid_for(l.rows * (l.kp / 8));
  const float e = ldexpf(1.0f, scale_exp);
  if (fmt == SCMP_MXFP4)
    mx_dequantize_kernel<T, SCMP_MXFP4><<<grid, kThreads, 0, s>>>(
        data, scales, l.rows, l.K, l.kp, l.groups, e, static_cast<T *>(out));
  else
    mx_dequantize_kernel<T, SCMP_NVFP4><<<grid, kThreads, 0, s>>>(
        data, scales, l.rows, l.K, l.kp, l.groups, e, static_cast<T *>(out));
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mx_quantize(const void *x, int dtype, int64_t ld, const MxLayout &l, int fmt,
                               int scale_exp, uint8_t *data, uint8_t *scales, cudaStream_t s,
                               int *launches) {
  *launches = 1;
  const bool mx = fmt == SCMP_MXFP4;
  if (dtype == SCMP_F32)
    return mx ? quantize<float, SCMP_MXFP4>(x, ld, l, scale_exp, data, scales, s)
              : quantize<float, SCMP_NVFP4>(x, ld, l, scale_exp, data, scales, s);
  if (dtype == SCMP_BF16)
    return mx ? quantize<__nv_bfloat16, SCMP_MXFP4>(x, ld, l, scale_exp, data, scales, s)
              : quantize<__nv_bfloat16, SCMP_NVFP4>(x, ld, l, scale_exp, data, scales, s);
  return mx ? quantize<__half, SCMP_MXFP4>(x, ld, l, scale_exp, data, scales, s)
            : quantize<__half, SCMP_NVFP4>(x, ld, l, scale_exp, data, scales, s);
}

cudaError_t launch_mx_dequantize(const uint8_t *data, const uint8_t *scales, const MxLayout &l,
                                 int fmt, int scale_exp, void *out, int dtype, cudaStream_t s) {
  if (dtype == SCMP_F32)
    return dequantize<float>(data, scales, l, fmt, scale_exp, out, s);
  if (dtype == SCMP_BF16)
    return dequantize<__nv_bfloat16>(data, scales, l, fmt, scale_exp, out, s);
  return dequantize<__half>(data, scales, l, fmt, scale_exp, out, s);
}

}  // namespace scmp
