// Quantisation to microscaled 4-bit floating point and back.
#include <cstring>

#include "mx_common.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;

constexpr int kAtOnce = 4;  // units in flight per warp: their loads are issued together

// Eight consecutive elements of a row at column k (those at or past K are 0).
template <typename T> struct Eight {
  uint4 u[sizeof(T) == 4 ? 2 : 1];
};
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T *__restrict__ row, int64_t k, int64_t K, bool live,
                                      Eight<T> &e) {
  if (kVec && live && k + 8 <= K) {
    const uint4 *p = reinterpret_cast<const uint4 *>(row + k);
    e.u[0] = __ldg(p);
    if (sizeof(T) == 4) e.u[sizeof(T) / 4] = __ldg(p + 1);
    return;
  }
  T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = live && k + i < K ? row[k + i] : from_f32<T>(0.0f);
  memcpy(&e, v, sizeof(e));
}

// Largest magnitude of eight elements, as the bits of an fp32 number.
template <typename T>
__device__ __forceinline__ uint32_t max_bits8(const Eight<T> &e, const float *v) {
  if (sizeof(T) == 4 || !__is_same(T, __nv_bfloat16)) return max_bits<8>(v);
  // bf16: two at a time, as 16-bit integers
  uint32_t m = __vmaxu2(__vmaxu2(e.u[0].x & 0x7FFF7FFFu, e.u[0].y & 0x7FFF7FFFu),
                        __vmaxu2(e.u[0].z & 0x7FFF7FFFu, e.u[0].w & 0x7FFF7FFFu));
  m = max(m >> 16, m & 0xFFFFu);
  return m << 16;
}

// A unit is 256 columns of one row, one warp: a lane holds eight consecutive
// values, the block's largest magnitude is a maximum over 4 (mxfp4) or 2
// (nvfp4) lanes, every lane stores 4 bytes of codes and a block's first lane its
// scale.  HBM-bound: FIXME.
template <typename T, int kFmt, bool kVec, bool kExp>
__global__ void __launch_bounds__(kThreads)
    mx_quantize_kernel(const T *__restrict__ x, int64_t ld, int64_t rows, int64_t K, int64_t kp,
                       int64_t groups, const __grid_constant__ FastDiv chunks, uint32_t units,
                       float inv_exp, uint8_t *__restrict__ data, uint8_t *__restrict__ scales) {
  constexpr int kLanes = kFmt == SCMP_MXFP4 ? 4 : 2;  // lanes per block
  const int lane = threadIdx.x & 31;
  const uint32_t warp = (blockIdx.x * kThreads + threadIdx.x) >> 5;
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint64_t u0 = (uint64_t)warp * kAtOnce; u0 < units; u0 += (uint64_t)warps * kAtOnce) {
    Eight<T> e[kAtOnce];
    uint32_t r[kAtOnce], k[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t u = (uint32_t)u0 + i;
      r[i] = chunks.quotient(u);
      k[i] = (u - r[i] * chunks.d) * 256 + lane * 8;
      load8<T, kVec>(x + r[i] * ld, k[i], K, u0 + i < units && r[i] < rows, e[i]);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (u0 + i >= units) break;
      float v[8];
      unpack16<T>(e[i].u[0], v);
      if (sizeof(T) == 4) unpack16<T>(e[i].u[sizeof(T) / 4], v + 4);
      uint32_t amax = max_bits8<T>(e[i], v), codes;
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) amax = max(amax, __shfl_xor_sync(~0u, amax, o));
      const uint32_t scale = mx_encode8<kFmt, kExp>(v, amax, inv_exp, &codes);
      if (r[i] < rows && k[i] < kp)
        *reinterpret_cast<uint32_t *>(data + r[i] * (kp >> 1) + (k[i] >> 1)) = codes;
      const uint32_t b = k[i] / (8 * kLanes);
      if ((lane & (kLanes - 1)) == 0 && (b >> 2) < groups)
        scales[mx_scale_word(r[i], b >> 2, groups) + (b & 3)] = (uint8_t)scale;
    }
  }
}

// Four (fp32) or eight (16-bit) consecutive elements per lane: 16 bytes out.
template <typename T, int kFmt>
__global__ void __launch_bounds__(kThreads)
    mx_dequantize_kernel(const uint8_t *__restrict__ data, const uint8_t *__restrict__ scales,
                         int64_t rows, int64_t K, int64_t kp, int64_t groups,
                         const __grid_constant__ FastDiv chunks, uint32_t units, float exp_value,
                         bool vec, T *__restrict__ out) {
  constexpr int kBlock = kFmt == SCMP_MXFP4 ? 32 : 16;
  constexpr int V = kVec16<T>;
  const int lane = threadIdx.x & 31;
  const uint32_t warp = (blockIdx.x * kThreads + threadIdx.x) >> 5;
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint64_t u0 = (uint64_t)warp * kAtOnce; u0 < units; u0 += (uint64_t)warps * kAtOnce) {
    uint32_t codes[kAtOnce], sc[kAtOnce], r[kAtOnce], k[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t u = (uint32_t)u0 + i;
      r[i] = chunks.quotient(u);
      k[i] = ((u - r[i] * chunks.d) * 32 + lane) * V;
      codes[i] = sc[i] = 0;
      if (u0 + i < units && k[i] < kp) {
        const uint8_t *src = data + r[i] * (kp >> 1) + (k[i] >> 1);
        codes[i] = V == 8 ? __ldg(reinterpret_cast<const uint32_t *>(src))
                          : __ldg(reinterpret_cast<const uint16_t *>(src));
        const uint32_t b = k[i] / kBlock;
        sc[i] = __ldg(scales + mx_scale_word(r[i], b >> 2, groups) + (b & 3));
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (u0 + i >= units || k[i] >= K) continue;
      float s;
      if (kFmt == SCMP_MXFP4)
        s = sc[i] == kMxNan ? __uint_as_float(0x7FC00000u) : e8m0_value(sc[i]);
      else
        s = e4m3_value(sc[i]) * exp_value;
      float v[V];
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        uint32_t h2;
        asm("{\n.reg .b8 b, z1, z2, z3;\nmov.b32 {b, z1, z2, z3}, %1;\n"
            "cvt.rn.f16x2.e2m1x2 %0, b;\n}\n"
            : "=r"(h2)
            : "r"(codes[i] >> (8 * j)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h2));
        v[2 * j] = f.x * s;
        v[2 * j + 1] = f.y * s;
      }
      T *dst = out + r[i] * K + k[i];
      if (vec) {
        *reinterpret_cast<uint4 *>(dst) = pack16<T>(v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (k[i] + j < K) dst[j] = from_f32<T>(v[j]);
      }
    }
  }
}

unsigned grid_for(uint32_t units) {
  const int64_t b = ((int64_t)units + kAtOnce * (kThreads / 32) - 1) / (kAtOnce * (kThreads / 32));
  return (unsigned)(b < 148 * 16 ? b : 148 * 16);
}

template <typename T, int kFmt, bool kVec>
cudaError_t quantize_v(const T *x, int64_t ld, const MxLayout &l, int scale_exp, uint8_t *data,
                       uint8_t *scales, cudaStream_t s) {
  const float inv_exp = ldexpf(1.0f, -scale_exp);
  // (rows and their 256-column units stay below 2^32 for what fits the memory)
  const FastDiv chunks((uint32_t)((l.kp + 255) / 256));
  const uint32_t units = (uint32_t)((l.rows + 127) / 128 * 128) * chunks.d;
  if (kFmt == SCMP_NVFP4 && scale_exp != 0)
    mx_quantize_kernel<T, kFmt, kVec, kFmt == SCMP_NVFP4><<<grid_for(units), kThreads, 0, s>>>(
        x, ld, l.rows, l.K, l.kp, l.groups, chunks, units, inv_exp, data, scales);
  else
    mx_quantize_kernel<T, kFmt, kVec, false><<<grid_for(units), kThreads, 0, s>>>(
        x, ld, l.rows, l.K, l.kp, l.groups, chunks, units, inv_exp, data, scales);
  return cudaGetLastError();
}
template <typename T, int kFmt>
cudaError_t quantize(const void *x, int64_t ld, const MxLayout &l, int scale_exp, uint8_t *data,
                     uint8_t *scales, cudaStream_t s) {
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
  const T *xt = static_cast<const T *>(x);
  return vec ? quantize_v<T, kFmt, true>(xt, ld, l, scale_exp, data, scales, s)
             : quantize_v<T, kFmt, false>(xt, ld, l, scale_exp, data, scales, s);
}

template <typename T>
cudaError_t dequantize(const uint8_t *data, const uint8_t *scales, const MxLayout &l, int fmt,
                       int scale_exp, void *out, cudaStream_t s) {
  constexpr int V = kVec16<T>;
  const FastDiv chunks((uint32_t)((l.kp + 32 * V - 1) / (32 * V)));
  const uint32_t units = (uint32_t)l.rows * chunks.d;
  const unsigned grid = grid_for(units);
  const bool vec = l.K % V == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const float e = ldexpf(1.0f, scale_exp);
  if (fmt == SCMP_MXFP4)
    mx_dequantize_kernel<T, SCMP_MXFP4><<<grid, kThreads, 0, s>>>(
        data, scales, l.rows, l.K, l.kp, l.groups, chunks, units, e, vec, static_cast<T *>(out));
  else
    mx_dequantize_kernel<T, SCMP_NVFP4><<<grid, kThreads, 0, s>>>(
        data, scales, l.rows, l.K, l.kp, l.groups, chunks, units, e, vec, static_cast<T *>(out));
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
