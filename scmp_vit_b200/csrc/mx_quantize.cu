// Quantisation to microscaled 4-bit floating point and back.
#include <cstring>

#include "mx_common.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;

// Eight consecutive elements per lane of a 256-column chunk of a row; those at
// or past K are 0.  Rows that are not made of 16-byte pieces are loaded one
// element per lane at a time, 32 neighbours, and dealt out through shared memory.
template <typename T, bool kVec> struct Chunk;
template <typename T> struct Chunk<T, true> {
  uint4 u[sizeof(T) == 4 ? 2 : 1];
  // k: the chunk's first column
  __device__ __forceinline__ void load(const T *row, int64_t k, int lane, int64_t K, bool live) {
    const T *p = row + k + lane * 8;
    k += lane * 8;
    if (live && k + 8 <= K) {
      u[0] = __ldg(reinterpret_cast<const uint4 *>(p));
      if (sizeof(T) == 4) u[sizeof(T) / 4] = __ldg(reinterpret_cast<const uint4 *>(p) + 1);
      return;
    }
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = live && k + i < K ? p[i] : from_f32<T>(0.0f);
    memcpy(u, v, sizeof(u));
  }
  __device__ __forceinline__ void deal(T *, int) {}
};
template <typename T> struct Chunk<T, false> {
  uint4 u[sizeof(T) == 4 ? 2 : 1];
  T raw[8];
  __device__ __forceinline__ void load(const T *row, int64_t k, int lane, int64_t K, bool live) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t c = k + lane + 32 * i;
      raw[i] = live && c < K ? row[c] : from_f32<T>(0.0f);
    }
  }
  __device__ __forceinline__ void deal(T *buf, int lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) buf[lane + 32 * i] = raw[i];
    __syncwarp();
    u[0] = reinterpret_cast<const uint4 *>(buf + lane * 8)[0];
    if (sizeof(T) == 4) u[sizeof(T) / 4] = reinterpret_cast<const uint4 *>(buf + lane * 8)[1];
    __syncwarp();
  }
};

// Largest magnitude of eight elements, as the bits of an fp32 number.
template <typename T>
__device__ __forceinline__ uint32_t max_bits8(const uint4 &u, const float *v) {
  if (!__is_same(T, __nv_bfloat16)) return max_bits<8>(v);
  // bf16: two at a time, as 16-bit integers
  uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu),
                        __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
  m = max(m >> 16, m & 0xFFFFu);
  return m << 16;
}

// A unit is kChunks x 256 columns of one row, one warp: a lane holds eight
// consecutive values of each chunk (all loads first), a block's largest
// magnitude is a maximum over 4 (mxfp4) or 2 (nvfp4) lanes, every lane stores 4
// bytes of codes and a block's first lane its scale.  The addresses of a unit
// are computed once: instructions, not only HBM, bound the 16-bit types (with
// addresses per chunk bf16 [32896, 4096] took 82 us, now 59: 5.8 TB/s).
template <typename T, int kFmt, bool kVec, bool kExp, int kChunks>
__global__ void __launch_bounds__(kThreads)
    mx_quantize_kernel(const T *__restrict__ x, int64_t ld, int64_t rows, int64_t K, int64_t kp,
                       int64_t groups, const __grid_constant__ FastDiv per_row, uint32_t units,
                       float inv_exp, uint8_t *__restrict__ data, uint8_t *__restrict__ scales) {
  constexpr int kLanes = kFmt == SCMP_MXFP4 ? 4 : 2;   // lanes per block
  constexpr int kGroups = 8 / kLanes;                  // scale groups per chunk
  __shared__ __align__(16) T deal[kVec ? 8 : kThreads * 8];
  // (a product behind this launch may set up as SMs become free)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  T *const buf = deal + (kVec ? 0 : (threadIdx.x >> 5) * 256);
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint64_t u = (blockIdx.x * kThreads + threadIdx.x) >> 5; u < units; u += warps) {
    const uint32_t r = per_row.quotient((uint32_t)u);
    const uint32_t chunk0 = ((uint32_t)u - r * per_row.d) * kChunks;
    const int64_t k = (int64_t)chunk0 * 256 + lane * 8;
    const bool live = r < rows;
    const T *row = x + r * ld;
    uint8_t *codes_at = data + r * (kp >> 1) + (k >> 1);
    const int b = lane / kLanes;  // block of the chunk
    const int64_t g = (int64_t)chunk0 * kGroups + (b >> 2);
    uint8_t *scale_at = scales + mx_scale_word(r, g, groups) + (b & 3);
    const bool first = (lane & (kLanes - 1)) == 0;
    Chunk<T, kVec> e[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) e[i].load(row, (int64_t)(chunk0 + i) * 256, lane, K, live);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      if (kChunks > 1 && (chunk0 + i) * 256 >= kp) break;
      e[i].deal(buf, lane);
      float v[8];
      unpack16<T>(e[i].u[0], v);
      if (sizeof(T) == 4) unpack16<T>(e[i].u[sizeof(T) / 4], v + 4);
      uint32_t amax = max_bits8<T>(e[i].u[0], v), codes;
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) amax = max(amax, __shfl_xor_sync(~0u, amax, o));
      const uint32_t scale = mx_encode8<kFmt, kExp>(v, amax, inv_exp, &codes);
      if (live && k + i * 256 < kp) *reinterpret_cast<uint32_t *>(codes_at + i * 128) = codes;
      if (first && g + i * kGroups < groups) scale_at[i * kGroups * 512] = (uint8_t)scale;
    }
  }
}

// Four (fp32) or eight (16-bit) consecutive elements per lane and chunk: 16
// bytes out, through shared memory and 32 neighbours at a time where rows are
// not made of such pieces.
template <typename T, int kFmt, int kChunks, bool kVec>
__global__ void __launch_bounds__(kThreads)
    mx_dequantize_kernel(const uint8_t *__restrict__ data, const uint8_t *__restrict__ scales,
                         int64_t rows, int64_t K, int64_t kp, int64_t groups,
                         const __grid_constant__ FastDiv per_row, uint32_t units, float exp_value,
                         T *__restrict__ out) {
  constexpr int kBlock = kFmt == SCMP_MXFP4 ? 32 : 16;
  constexpr int V = kVec16<T>;
  __shared__ __align__(16) T deal[kVec ? 8 : kThreads * V];
  const int lane = threadIdx.x & 31;
  T *const buf = deal + (kVec ? 0 : (threadIdx.x >> 5) * 32 * V);
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint64_t u = (blockIdx.x * kThreads + threadIdx.x) >> 5; u < units; u += warps) {
    const uint32_t r = per_row.quotient((uint32_t)u);
    const int64_t k = ((int64_t)((uint32_t)u - r * per_row.d) * kChunks * 32 + lane) * V;
    const uint8_t *src = data + r * (kp >> 1) + (k >> 1);
    uint32_t codes[kChunks], sc[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      codes[i] = sc[i] = 0;
      const int64_t ki = k + i * 32 * V;
      if (ki < kp) {
        codes[i] = V == 8 ? __ldg(reinterpret_cast<const uint32_t *>(src + i * 16 * V))
                          : __ldg(reinterpret_cast<const uint16_t *>(src + i * 16 * V));
        const int64_t b = ki / kBlock;
        sc[i] = __ldg(scales + mx_scale_word(r, b >> 2, groups) + (b & 3));
      }
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int64_t ki = k + i * 32 * V;
      if (ki - lane * V >= K) break;
      float s;
      if (kFmt == SCMP_MXFP4)
        s = sc[i] == kMxNan ? __uint_as_float(0x7FC00000u) : e8m0_value(sc[i]);
      else
        s = e4m3_value(sc[i]);
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
        if (kFmt == SCMP_NVFP4) {
          // last, since a scale times the tensor's may leave fp32's range where
          // the value, a zero's for one, does not
          v[2 * j] *= exp_value;
          v[2 * j + 1] *= exp_value;
        }
      }
      T *dst = out + r * K + ki;
      if (kVec) {
        if (ki < K) *reinterpret_cast<uint4 *>(dst) = pack16<T>(v);
      } else {
        *reinterpret_cast<uint4 *>(buf + lane * V) = pack16<T>(v);
        __syncwarp();
        const int64_t c = ki - lane * V + lane;  // a neighbour per lane
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + 32 * j < K) out[r * K + c + 32 * j] = buf[lane + 32 * j];
        __syncwarp();
      }
    }
  }
}

unsigned grid_for(uint32_t units) {
  const int64_t b = ((int64_t)units + kThreads / 32 - 1) / (kThreads / 32);
  return (unsigned)(b < 148 * 16 ? b : 148 * 16);
}

// (rows and their units stay below 2^32 for what fits the memory)
template <typename T, int kFmt, bool kVec, bool kExp, int kChunks>
cudaError_t quantize_k(const T *x, int64_t ld, const MxLayout &l, float inv_exp, uint8_t *data,
                       uint8_t *scales, cudaStream_t s) {
  const FastDiv per_row((uint32_t)((l.kp + 256 * kChunks - 1) / (256 * kChunks)));
  const uint32_t units = (uint32_t)((l.rows + 127) / 128 * 128) * per_row.d;
  mx_quantize_kernel<T, kFmt, kVec, kExp, kChunks><<<grid_for(units), kThreads, 0, s>>>(
      x, ld, l.rows, l.K, l.kp, l.groups, per_row, units, inv_exp, data, scales);
  return cudaGetLastError();
}
template <typename T, int kFmt, bool kVec, bool kExp>
cudaError_t quantize_e(const T *x, int64_t ld, const MxLayout &l, float inv_exp, uint8_t *data,
                       uint8_t *scales, cudaStream_t s) {
  // four chunks in flight per warp; one for short rows and where there would be
  // fewer than eight warps on each of the 148 SMs
  const int64_t units = l.rows * ((l.kp + 1023) / 1024);
  return l.kp <= 512 || units < 148 * 8
             ? quantize_k<T, kFmt, kVec, kExp, 1>(x, ld, l, inv_exp, data, scales, s)
             : quantize_k<T, kFmt, kVec, kExp, 4>(x, ld, l, inv_exp, data, scales, s);
}
template <typename T, int kFmt, bool kVec>
cudaError_t quantize_v(const T *x, int64_t ld, const MxLayout &l, int scale_exp, uint8_t *data,
                       uint8_t *scales, cudaStream_t s) {
  const float inv_exp = ldexpf(1.0f, -scale_exp);
  if (kFmt == SCMP_NVFP4 && scale_exp != 0)
    return quantize_e<T, kFmt, kVec, kFmt == SCMP_NVFP4>(x, ld, l, inv_exp, data, scales, s);
  return quantize_e<T, kFmt, kVec, false>(x, ld, l, inv_exp, data, scales, s);
}
template <typename T, int kFmt>
cudaError_t quantize(const void *x, int64_t ld, const MxLayout &l, int scale_exp, uint8_t *data,
                     uint8_t *scales, cudaStream_t s) {
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
  const T *xt = static_cast<const T *>(x);
  return vec ? quantize_v<T, kFmt, true>(xt, ld, l, scale_exp, data, scales, s)
             : quantize_v<T, kFmt, false>(xt, ld, l, scale_exp, data, scales, s);
}

template <typename T, int kFmt, int kChunks, bool kVec>
cudaError_t dequantize_v(const uint8_t *data, const uint8_t *scales, const MxLayout &l,
                         int scale_exp, void *out, cudaStream_t s) {
  constexpr int V = kVec16<T>;
  const FastDiv per_row((uint32_t)((l.kp + 32 * V * kChunks - 1) / (32 * V * kChunks)));
  const uint32_t units = (uint32_t)l.rows * per_row.d;
  mx_dequantize_kernel<T, kFmt, kChunks, kVec><<<grid_for(units), kThreads, 0, s>>>(
      data, scales, l.rows, l.K, l.kp, l.groups, per_row, units, ldexpf(1.0f, scale_exp),
      static_cast<T *>(out));
  return cudaGetLastError();
}
template <typename T, int kFmt, int kChunks>
cudaError_t dequantize_k(const uint8_t *data, const uint8_t *scales, const MxLayout &l,
                         int scale_exp, void *out, cudaStream_t s) {
  const bool vec = l.K % kVec16<T> == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  return vec ? dequantize_v<T, kFmt, kChunks, true>(data, scales, l, scale_exp, out, s)
             : dequantize_v<T, kFmt, kChunks, false>(data, scales, l, scale_exp, out, s);
}
template <typename T>
cudaError_t dequantize(const uint8_t *data, const uint8_t *scales, const MxLayout &l, int fmt,
                       int scale_exp, void *out, cudaStream_t s) {
  const int64_t chunk = 32 * kVec16<T>, units = l.rows * ((l.kp + 4 * chunk - 1) / (4 * chunk));
  const bool one = l.kp <= 2 * chunk || units < 148 * 8;  // as in quantize_e
  if (fmt == SCMP_MXFP4)
    return one ? dequantize_k<T, SCMP_MXFP4, 1>(data, scales, l, scale_exp, out, s)
               : dequantize_k<T, SCMP_MXFP4, 4>(data, scales, l, scale_exp, out, s);
  return one ? dequantize_k<T, SCMP_NVFP4, 1>(data, scales, l, scale_exp, out, s)
             : dequantize_k<T, SCMP_NVFP4, 4>(data, scales, l, scale_exp, out, s);
}

}  // namespace

cudaError_t launch_mx_quantize(const void *x, int dtype, int64_t ld, const MxLayout &l, int fmt,
                               int scale_exp, uint8_t *data, uint8_t *scales, cudaStream_t s) {
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
