// Device pieces of the qkv splits (rotary.cu, qknorm.cu): vector pieces of a head
// row, a token's cos and sin, the transposed tiles of v.  Internal linkage.
#pragma once

#include <cstring>

#include "mx_common.cuh"
#include "rotary.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;  // tokens of a transposed tile

// V elements as loaded: 16, 8 or 4 bytes, or one element.
template <typename T, int V> struct Piece {
  static constexpr int kWords = V * (int)sizeof(T) / 4;
  uint32_t u[kWords];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (kWords == 4)
      *reinterpret_cast<uint4 *>(u) = *reinterpret_cast<const uint4 *>(p);
    else if constexpr (kWords == 2)
      *reinterpret_cast<uint2 *>(u) = *reinterpret_cast<const uint2 *>(p);
    else
      u[0] = *reinterpret_cast<const uint32_t *>(p);
  }
  __device__ __forceinline__ void store(T *p) const {
    if constexpr (kWords == 4)
      *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(u);
    else if constexpr (kWords == 2)
      *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(u);
    else
      *reinterpret_cast<uint32_t *>(p) = u[0];
  }
  __device__ __forceinline__ void get(float *v) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(u[i]);
      } else {
        const float2 f = unpack2<T>(u[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
  // word i from its elements v
  static __device__ __forceinline__ uint32_t word(const float *v, int i) {
    if constexpr (sizeof(T) == 4)
      return __float_as_uint(v[i]);
    else
      return pack2<T>(v[2 * i], v[2 * i + 1]);
  }
};
template <typename T> struct Piece<T, 1> {
  T u[1];
  __device__ __forceinline__ void load(const T *p) { u[0] = *p; }
  __device__ __forceinline__ void store(T *p) const { *p = u[0]; }
};

// cos and signed sin of V elements of a token's head from e0 on, the bits of
// those that turn and the first one's partner.  A negative coordinate leaves its
// axis as it is, one past the table's end gives NaN rather than a read there.
template <int V, bool kInterleaved, bool kBackward>
__device__ __forceinline__ uint32_t angles_of(const RotaryParams &p, int64_t token, int e0,
                                              float (&c)[V], float (&s)[V], int &partner) {
  uint32_t mask = 0;
  partner = e0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    c[j] = 1.0f;
    s[j] = 0.0f;
  }
  // sections are walked, not searched per element: a piece touches one or two
  int end = 0;
#pragma unroll
  for (int a = 0; a < SCMP_MAX_AXES; ++a) {
    if (a >= p.axes) break;
    const int begin = end, half = p.dims[a] >> 1;
    end += p.dims[a];
    if (e0 >= end || e0 + V <= begin) continue;
    const int coord = p.pos[token * p.axes + a];
    const bool second0 = !kInterleaved && e0 - begin >= half;  // (a piece has one half, V > 1)
    if (e0 >= begin) partner = kInterleaved ? e0 ^ 1 : second0 ? e0 - half : e0 + half;
    if (coord < 0) continue;
    const float2 *row = p.table + p.table_at[a] + (int64_t)coord * half;
    const bool known = coord < p.sizes[a];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int o = e0 + j - begin;
      if (o < 0 || e0 + j >= end) continue;
      if (kInterleaved && V > 1 && (o & 1)) continue;  // set with the pair's first member
      const int i = kInterleaved ? o >> 1 : second0 ? o - half : o;
      float2 cs = make_float2(__uint_as_float(0x7FC00000u), __uint_as_float(0x7FC00000u));
      if (known) cs = __ldg(row + i);
      // the first member of a pair subtracts (adds, going back)
      if (kInterleaved && V > 1) {
        c[j] = cs.x;
        s[j] = kBackward ? cs.y : -cs.y;
        if (j + 1 < V) {
          c[j + 1] = cs.x;
          s[j + 1] = -s[j];
        }
        mask |= 3u << j;
      } else {
        const bool second = kInterleaved ? (o & 1) : second0;
        c[j] = cs.x;
        s[j] = second != kBackward ? cs.y : -cs.y;
        mask |= 1u << j;
      }
    }
  }
  return mask;
}

// v of one head, kTile tokens: token rows of the fused tensor <-> [D, N], through
// a tile [D][kTile + 2].  Global accesses go in batches of kBatch per thread
// (one at a time, 64 images in bf16 took 96 us, now 50).
constexpr int kBatch = 4;
template <typename T, int V, bool kBackward>
__device__ __forceinline__ void transpose_tile(const RotaryParams &p, uint32_t block, T *tile) {
  constexpr int kPitch = kTile + 2;
  const uint32_t tiles = (uint32_t)((p.N + kTile - 1) / kTile);
  const int64_t bh = block / tiles, b = bh / p.Hk, h = bh % p.Hk;
  const int64_t t0 = (int64_t)(block % tiles) * kTile;
  const int nt = (int)(p.N - t0 < kTile ? p.N - t0 : kTile);
  const int D = p.D, per = D / V;
  const int64_t step = (p.H + 2 * p.Hk) * D;
  T *const fused = static_cast<T *>(p.qkv) + ((b * p.N + t0) * step + (p.H + p.Hk + h) * D);
  T *const flat = static_cast<T *>(p.v) + bh * D * p.N + t0;
  const int pieces = nt * per, elems = D * kTile;  // (lanes of a [D, N] row: kTile at a time)
  if (!kBackward) {
    for (int i0 = threadIdx.x; i0 < pieces; i0 += kThreads * kBatch) {
      Piece<T, V> x[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = i0 + k * kThreads;
        if (i < pieces) x[k].load(fused + i / per * step + i % per * V);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = i0 + k * kThreads;
        if (i >= pieces) break;
        T v[V];
        memcpy(v, x[k].u, sizeof(v));
#pragma unroll
        for (int j = 0; j < V; ++j) tile[(i % per * V + j) * kPitch + i / per] = v[j];
      }
    }
  } else {
    for (int i0 = threadIdx.x; i0 < elems; i0 += kThreads * 2 * kBatch) {
      T x[2 * kBatch];
#pragma unroll
      for (int k = 0; k < 2 * kBatch; ++k) {
        const int i = i0 + k * kThreads, t = i % kTile;
        if (i < elems && t < nt) x[k] = flat[(int64_t)(i / kTile) * p.N + t];
      }
#pragma unroll
      for (int k = 0; k < 2 * kBatch; ++k) {
        const int i = i0 + k * kThreads, t = i % kTile;
        if (i < elems && t < nt) tile[i / kTile * kPitch + t] = x[k];
      }
    }
  }
  __syncthreads();
  if (kBackward) {
    for (int i = threadIdx.x; i < pieces; i += kThreads) {
      T v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = tile[(i % per * V + j) * kPitch + i / per];
      Piece<T, V> x;
      memcpy(x.u, v, sizeof(v));
      x.store(fused + i / per * step + i % per * V);
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < elems; i += kThreads) {
      const int t = i % kTile;
      if (t < nt) flat[(int64_t)(i / kTile) * p.N + t] = tile[i / kTile * kPitch + t];
    }
  }
}

// Whether pieces of V elements divide every head row and, with the two members
// of a pair half a section apart, every half section (a piece's partners are
// then a piece).  (t, h, w) sections of 16, 24, 24 take 8 bytes of 16-bit types.
template <typename T, int V> bool pieces(const RotaryParams &p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.qkv) | reinterpret_cast<uintptr_t>(p.q) |
                       reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
  bool ok = p.D % V == 0 && at % (V * sizeof(T)) == 0;
  if (!p.interleaved)
    for (int a = 0; a < p.axes; ++a) ok = ok && (p.dims[a] / 2) % V == 0;
  return ok;
}

}  // namespace
}  // namespace scmp
