// Rows of fp32, bf16 or fp16 on their way into codes: pieces of 256 columns, one
// warp each (internal).
#pragma once

#include <cstring>

#include "mx_common.cuh"

namespace scmp {

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

}  // namespace scmp
