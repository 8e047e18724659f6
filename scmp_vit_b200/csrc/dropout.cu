// Dropout from a counter-based generator, with an optional residual add:
//   y[i] = residual[i] + (u_d < p 2^32 ? 0 : x[i] / (1 - p)),   d = i / span,
// u_d = word d % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random
// numbers: as easy as 1, 2, 3, 2011) at counter (d / 4, offset) under the key `seed`.
// No mask is stored: the backward pass calls the same kernel on the gradient and
// draws the same words.
//
// span 1: a thread takes eight consecutive elements, two blocks of the generator
// (40 wide multiplications), which HBM hides: 16-byte loads, one launch, each
// element read and written once.  Longer spans draw once per piece of elements.
#include "dropout.cuh"

#include "mx_common.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;

// Philox4x32-10: ten rounds of two 32 x 32 -> 64 bit products, the key stepped by
// Weyl constants.
__device__ __forceinline__ uint4 philox(uint64_t counter, uint64_t offset, uint64_t key) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = (uint32_t)offset,
           c3 = (uint32_t)(offset >> 32), k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ uint32_t word(const uint4 &u, uint32_t i) {
  return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
}

// Dropped values are left out, not multiplied by 0: what a NaN or an infinity leaves
// there is 0.
__device__ __forceinline__ float one(float x, float residual, uint32_t u, const DropoutParams &p) {
  const float kept = u < p.threshold ? 0.0f : x * p.scale;
  return p.residual ? residual + kept : kept;
}

// Eight elements per thread and step; kVec: all pointers on 16 bytes (n need not be
// a multiple).
template <typename T, bool kVec, bool kSpan>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const __grid_constant__ DropoutParams p) {
  constexpr int kLoads = 8 / kVec16<T>;
  uint64_t seed = p.seed, offset = p.offset;
  if (p.state) {
    seed = p.state[0];
    offset += p.state[1];
  }
  const T *x = static_cast<const T *>(p.x), *residual = static_cast<const T *>(p.residual);
  T *y = static_cast<T *>(p.y);
  const int64_t step = (int64_t)gridDim.x * kThreads * 8;
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 8; i < p.n; i += step) {
    const bool whole = kVec && i + 8 <= p.n;
    float v[8], r[8];
    if (whole) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        // (plain loads: y may be x or residual)
        unpack16<T>(reinterpret_cast<const uint4 *>(x + i)[l], v + l * kVec16<T>);
        if (residual)
          unpack16<T>(reinterpret_cast<const uint4 *>(residual + i)[l], r + l * kVec16<T>);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = i + j < p.n ? to_f32(x[i + j]) : 0.0f;
        r[j] = residual && i + j < p.n ? to_f32(residual[i + j]) : 0.0f;
      }
    }
    if (!kSpan) {
      const uint4 a = philox((uint64_t)i >> 2, offset, seed);
      const uint4 b = philox(((uint64_t)i >> 2) + 1, offset, seed);
      const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = one(v[j], r[j], u[j], p);
    } else {
      uint64_t d = (uint64_t)i / (uint64_t)p.span, end = (d + 1) * (uint64_t)p.span;
      uint32_t u = word(philox(d >> 2, offset, seed), (uint32_t)d & 3);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if ((uint64_t)i + j == end) {
          ++d;
          end += (uint64_t)p.span;
          u = word(philox(d >> 2, offset, seed), (uint32_t)d & 3);
        }
        v[j] = one(v[j], r[j], u, p);
      }
    }
    if (whole) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l)
        reinterpret_cast<uint4 *>(y + i)[l] = pack16<T>(v + l * kVec16<T>);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < p.n) y[i + j] = from_f32<T>(v[j]);
    }
  }
}

template <typename T> cudaError_t launch(const DropoutParams &p, cudaStream_t s) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.residual) |
                       reinterpret_cast<uintptr_t>(p.y);
  const bool vec = at % 16 == 0, span = p.span > 1;
  const int64_t blocks = ((p.n + 7) / 8 + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16);
  if (vec)
    span ? dropout_kernel<T, true, true><<<grid, kThreads, 0, s>>>(p)
         : dropout_kernel<T, true, false><<<grid, kThreads, 0, s>>>(p);
  else
    span ? dropout_kernel<T, false, true><<<grid, kThreads, 0, s>>>(p)
         : dropout_kernel<T, false, false><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_dropout(const DropoutParams &p, int dtype, cudaStream_t s) {
  if (dtype == SCMP_F32) return launch<float>(p, s);
  if (dtype == SCMP_BF16) return launch<__nv_bfloat16>(p, s);
  return launch<__half>(p, s);
}

}  // namespace scmp
