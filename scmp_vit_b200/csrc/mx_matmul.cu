// Product of two microscaled 4-bit operands: out[m, n] = sum_k A[m, k] B[n, k]
// (+ bias[n]), A [M, K] and B [N, K] in the layout of mx_common.cuh.
#include "mx_common.cuh"

namespace scmp {
namespace {

// 32 x 32 output tile, 32 values of K at a time widened to fp32 in shared
// memory.
template <int kFmt>
__device__ __forceinline__ float mx_value(const uint8_t *data, const uint8_t *scales, int64_t r,
                                          int64_t k, int64_t kp, int64_t groups) {
  constexpr int kBlock = kFmt == SCMP_MXFP4 ? 32 : 16;
  const uint32_t code = (data[r * (kp >> 1) + (k >> 1)] >> (4 * (k & 1))) & 15u;
  const uint32_t m = code & 7u;
  const float mag = m < 4 ? 0.5f * (float)m : m < 6 ? (float)(m - 2) : (float)(2 * m - 8);
  const int64_t b = k / kBlock;
  const uint32_t sc = scales[mx_scale_word(r, b >> 2, groups) + (b & 3)];
  float s;
  if (kFmt == SCMP_MXFP4)
    s = sc == kMxNan ? __uint_as_float(0x7FC00000u) : e8m0_value(sc);
  else
    s = e4m3_value(sc);
  return (code & 8u ? -mag : mag) * s;
}

__device__ __forceinline__ float load_as_f32(const void *p, int dtype, int64_t i) {
  if (dtype == SCMP_F32) return static_cast<const float *>(p)[i];
  if (dtype == SCMP_BF16) return to_f32(static_cast<const __nv_bfloat16 *>(p)[i]);
  return to_f32(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void store_as(void *p, int dtype, int64_t i, float v) {
  if (dtype == SCMP_F32)
    static_cast<float *>(p)[i] = v;
  else if (dtype == SCMP_BF16)
    static_cast<__nv_bfloat16 *>(p)[i] = from_f32<__nv_bfloat16>(v);
  else
    static_cast<__half *>(p)[i] = from_f32<__half>(v);
}

template <int kFmt>
__global__ void __launch_bounds__(256) mx_matmul_kernel(const MxProduct p, int64_t kp,
                                                        int64_t groups, int64_t tiles_n) {
  __shared__ float a[32][33], b[32][33];
  const int64_t m0 = (blockIdx.x / tiles_n) * 32, n0 = (blockIdx.x % tiles_n) * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t k0 = 0; k0 < kp; k0 += 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = ty + 8 * i;
      a[r][tx] = m0 + r < p.M
                     ? mx_value<kFmt>(p.a, p.a_scales, m0 + r, k0 + tx, kp, groups) : 0.f;
      b[r][tx] = n0 + r < p.N
                     ? mx_value<kFmt>(p.b, p.b_scales, n0 + r, k0 + tx, kp, groups) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 32; ++k) acc[i] = __fmaf_rn(a[ty + 8 * i][k], b[tx][k], acc[i]);
    __syncthreads();
  }
  const int64_t n = n0 + tx;
  if (n >= p.N) return;
  const float bias = p.bias ? load_as_f32(p.bias, p.bias_dtype, n) : 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 8 * i;
    if (m < p.M)
      store_as(p.out, p.out_dtype, m * p.N + n,
               p.bias ? __fmaf_rn(acc[i], p.alpha, bias) : acc[i] * p.alpha);
  }
}

}  // namespace

cudaError_t launch_mx_matmul(const MxProduct &p, unsigned int *error, cudaStream_t s,
                             int *launches) {
  (void)error;
  *launches = 1;
  const MxLayout l = mx_layout(p.M, p.K, p.fmt);
  const int64_t tm = (p.M + 31) / 32, tn = (p.N + 31) / 32;
  if (p.fmt == SCMP_MXFP4)
    mx_matmul_kernel<SCMP_MXFP4><<<(unsigned)(tm * tn), 256, 0, s>>>(p, l.kp, l.groups, tn);
  else
    mx_matmul_kernel<SCMP_NVFP4><<<(unsigned)(tm * tn), 256, 0, s>>>(p, l.kp, l.groups, tn);
  return cudaGetLastError();
}

}  // namespace scmp
