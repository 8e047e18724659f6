// Dropout from a counter-based generator, with an optional residual add:
//   y[i] = residual[i] + (u_d < p 2^32 ? 0 : x[i] / (1 - p)),   d = i / span,
// u_d = word d % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random
// numbers: as easy as 1, 2, 3, 2011) at counter (d / 4, offset) under the key `seed`.
// No mask is stored: the backward pass calls the same kernel on the gradient and
// draws the same words.
//
// A thread takes eight consecutive elements: 16-byte loads, one launch, each element
// read and written once.  With spans of many elements that is bound by HBM: bf16
// [64, 257, 4096] per sample 43 us, a copy of it 42.6; fp32 per element 84 us (6.4 TB/s).
// 16-bit elements that all draw are bound by instructions: two blocks of the generator
// (40 wide multiplications) for 32 bytes moved, 59 us, with a residual 64.
#include "dropout.cuh"

#include <cstring>

#include "mx_common.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;

// Ten rounds of two 32 x 32 -> 64 bit products.  The rounds' keys (Weyl steps of the
// seed) come ready made, from the kernel's arguments where the seed does: added up
// in every round they were a third of the kernel's integer work.
template <typename I>
__device__ __forceinline__ uint4 philox(I counter, uint64_t offset, const uint32_t *keys) {
  uint32_t c0 = (uint32_t)counter, c1 = sizeof(I) == 8 ? (uint32_t)((uint64_t)counter >> 32) : 0u,
           c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ keys[2 * r];
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ keys[2 * r + 1];
    c3 = (uint32_t)a;
  }
  return make_uint4(c0, c1, c2, c3);
}
__host__ __device__ inline void round_keys(uint64_t seed, uint32_t *keys) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    keys[2 * r] = (uint32_t)seed + 0x9E3779B9u * (uint32_t)r;
    keys[2 * r + 1] = (uint32_t)(seed >> 32) + 0xBB67AE85u * (uint32_t)r;
  }
}
__device__ __forceinline__ uint32_t word(const uint4 &u, uint32_t i) {
  return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
}

// Dropped values are left out, not multiplied by 0: what a NaN or an infinity leaves
// there is 0.
__device__ __forceinline__ float kept(float x, uint32_t u, const DropoutParams &p) {
  return u > p.limit ? x * p.scale : 0.0f;
}

// Eight elements as loaded; kVec: all pointers on 16 bytes.
template <typename T, bool kVec> struct Eight {
  static constexpr int kLoads = 8 / kVec16<T>;
  uint4 u[kLoads];
  // (plain loads: y may be x or residual)
  __device__ __forceinline__ void load(const T *p, int64_t left) {
    if (kVec && left >= 8) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) u[l] = reinterpret_cast<const uint4 *>(p)[l];
    } else {
      T e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = j < left ? p[j] : from_f32<T>(0.0f);
      memcpy(u, e, sizeof(u));
    }
  }
  __device__ __forceinline__ void store(T *p, int64_t left) const {
    if (kVec && left >= 8) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) reinterpret_cast<uint4 *>(p)[l] = u[l];
    } else {
      T e[8];
      memcpy(e, u, sizeof(u));
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) p[j] = e[j];
    }
  }
};

// i / span: 64-bit divisions cost more than a block of the generator.
__device__ __forceinline__ uint32_t quotient(const DropoutParams &p, uint32_t i) {
  return p.per_span.quotient(i);
}
__device__ __forceinline__ uint64_t quotient(const DropoutParams &p, uint64_t i) {
  return i / (uint64_t)p.span;
}

// The draws of eight elements from i on; `last` and `w` are a span and its draw, the
// last ones used.
template <int kDraw, typename I>
__device__ __forceinline__ void draws(const DropoutParams &p, I i, uint64_t offset,
                                      const uint32_t *keys, I &last, uint32_t &w,
                                      uint32_t (&u)[8]) {
  if (kDraw == 1) {
    const uint4 a = philox<I>(i >> 2, offset, keys), b = philox<I>((i >> 2) + 1, offset, keys);
    u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w;
    u[4] = b.x; u[5] = b.y; u[6] = b.z; u[7] = b.w;
  } else if (kDraw == 2) {
    I d = quotient(p, i), end = (d + 1) * (I)p.span;
    if (d != last) w = word(philox<I>(d >> 2, offset, keys), (uint32_t)d & 3);
    if (i + 8 <= end) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (i + j == end) {
          ++d;
          end += (I)p.span;
          w = word(philox<I>(d >> 2, offset, keys), (uint32_t)d & 3);
        }
        u[j] = w;
      }
    }
    last = d;
  }
}

// steps() x 8 elements per thread, all loads first.  kDraw 0: nothing is dropped, 1: a
// draw per element, 2: per span.  Two steps for 16-bit types that HBM bounds (bf16 as
// above, per sample 43 us, with one step 58; per element 61, one 59; fp32 84 either way,
// [257, 1024] 2.0 and 1.7).
template <typename T, int kDraw> __host__ __device__ constexpr int steps() {
  return sizeof(T) == 2 && kDraw != 1 ? 2 : 1;
}
template <typename T, bool kVec, bool kResidual, int kDraw, bool kState, typename I>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const __grid_constant__ DropoutParams p) {
  constexpr int kSteps = steps<T, kDraw>();
  constexpr int64_t kBlock = kThreads * 8;
  uint64_t offset = p.offset;
  uint32_t own[20];
  if (kState) {
    round_keys(p.state[0], own);
    offset += p.state[1];
  }
  const T *x = static_cast<const T *>(p.x), *residual = static_cast<const T *>(p.residual);
  T *y = static_cast<T *>(p.y);
  I last = ~(I)0;
  uint32_t w = 0;
  for (int64_t i0 = blockIdx.x * kBlock * kSteps + threadIdx.x * 8; i0 < p.n;
       i0 += gridDim.x * kBlock * kSteps) {
    Eight<T, kVec> xs[kSteps], rs[kSteps];
#pragma unroll
    for (int q = 0; q < kSteps; ++q) {
      const int64_t i = i0 + q * kBlock;
      xs[q].load(x + i, p.n - i);
      if (kResidual) rs[q].load(residual + i, p.n - i);
    }
#pragma unroll
    for (int q = 0; q < kSteps; ++q) {
      const int64_t i = i0 + q * kBlock;
      if (i >= p.n) break;
      uint32_t u[8];
      draws<kDraw, I>(p, (I)i, offset, kState ? own : p.keys, last, w, u);
      float v[8], r[8];
#pragma unroll
      for (int l = 0; l < Eight<T, kVec>::kLoads; ++l) {
        unpack16<T>(xs[q].u[l], v + l * kVec16<T>);
        if (kResidual) unpack16<T>(rs[q].u[l], r + l * kVec16<T>);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = kDraw ? kept(v[j], u[j], p) : v[j] * p.scale;
        if (kResidual) v[j] = r[j] + v[j];
      }
#pragma unroll
      for (int l = 0; l < Eight<T, kVec>::kLoads; ++l) xs[q].u[l] = pack16<T>(v + l * kVec16<T>);
      xs[q].store(y + i, p.n - i);
    }
  }
}

template <typename T, bool kVec, bool kResidual, int kDraw, bool kState, typename I>
void launch_kernel(const DropoutParams &p, cudaStream_t s) {
  const int64_t per = kThreads * 8 * steps<T, kDraw>(), blocks = (p.n + per - 1) / per;
  const unsigned grid = (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16);
  dropout_kernel<T, kVec, kResidual, kDraw, kState, I><<<grid, kThreads, 0, s>>>(p);
}
template <typename T, bool kVec, bool kResidual, typename I>
void launch_draw(const DropoutParams &p, cudaStream_t s) {
  if (p.none)
    launch_kernel<T, kVec, kResidual, 0, false, I>(p, s);
  else if (p.span == 1 && !p.state)
    launch_kernel<T, kVec, kResidual, 1, false, I>(p, s);
  else if (p.span == 1)
    launch_kernel<T, kVec, kResidual, 1, true, I>(p, s);
  else if (!p.state)
    launch_kernel<T, kVec, kResidual, 2, false, I>(p, s);
  else
    launch_kernel<T, kVec, kResidual, 2, true, I>(p, s);
}
// Elements counted in 32 bits where they and the end of their last span fit.
template <typename T, bool kVec, bool kResidual>
void launch_index(DropoutParams p, cudaStream_t s) {
  if (p.n <= INT32_MAX && p.span <= INT32_MAX) {
    p.per_span = FastDiv((uint32_t)p.span);
    launch_draw<T, kVec, kResidual, uint32_t>(p, s);
  } else {
    launch_draw<T, kVec, kResidual, uint64_t>(p, s);
  }
}
template <typename T> cudaError_t launch(const DropoutParams &p, cudaStream_t s) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.residual) |
                       reinterpret_cast<uintptr_t>(p.y);
  const bool vec = at % 16 == 0;
  if (vec)
    p.residual ? launch_index<T, true, true>(p, s) : launch_index<T, true, false>(p, s);
  else
    p.residual ? launch_index<T, false, true>(p, s) : launch_index<T, false, false>(p, s);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_dropout(DropoutParams p, uint64_t seed, int dtype, cudaStream_t s) {
  round_keys(seed, p.keys);
  if (dtype == SCMP_F32) return launch<float>(p, s);
  if (dtype == SCMP_BF16) return launch<__nv_bfloat16>(p, s);
  return launch<__half>(p, s);
}

}  // namespace scmp
