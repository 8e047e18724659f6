// The fused qkv projection output split into q, k and v with q and k turned by
// multi-axis rotary positions, and its gradient.
//   pair (u, v) of axis a, frequency i, at coordinate c:
//     u' = u cos t - v sin t,  v' = v cos t + u sin t,  t = c scale_a base^(-2 i / d_a)
// cos and sin come from a table per axis (rows = coordinates), built in 64 bits
// where far coordinates need them; the backward pass turns by -t.
#include "rotary.cuh"

#include "mx_common.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 32;  // tokens per block

// cos and sin of every pair of a tile's tokens in shared memory, [kTile][pairs].
// A negative coordinate leaves the token's pairs of that axis as they are; one
// past the table's end makes them NaN rather than read there.
__device__ __forceinline__ void stage_angles(const RotaryParams &p, int64_t b, int64_t t0, int nt,
                                             float2 *cs) {
  const int pairs = p.pairs;
  for (int i = threadIdx.x; i < nt * pairs; i += kThreads) {
    const int t = i / pairs, q = i % pairs;
    int a = 0;
    while (a + 1 < p.axes && q >= p.first_pair[a + 1]) ++a;
    const int c = p.pos[((p.pos_batched ? b * p.N : 0) + t0 + t) * p.axes + a];
    const int half = p.dims[a] >> 1;
    float2 v = make_float2(1.0f, 0.0f);
    if (c >= p.sizes[a])
      v = make_float2(__uint_as_float(0x7FC00000u), __uint_as_float(0x7FC00000u));
    else if (c >= 0)
      v = p.table[p.table_at[a] + (int64_t)c * half + (q - p.first_pair[a])];
    if (p.inverse) v.y = -v.y;
    cs[i] = v;
  }
}

// Element index of the first and second member of pair q inside a head.
__device__ __forceinline__ int2 pair_at(const RotaryParams &p, int q) {
  int a = 0;
  while (a + 1 < p.axes && q >= p.first_pair[a + 1]) ++a;
  const int i = q - p.first_pair[a], base = 2 * p.first_pair[a];
  return p.interleaved ? make_int2(base + 2 * i, base + 2 * i + 1)
                       : make_int2(base + i, base + i + (p.dims[a] >> 1));
}

// One pair per thread; any alignment.
template <typename T, bool kBackward>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ float2 cs[];
  const int64_t tiles = (p.N + kTile - 1) / kTile;
  const int64_t b = blockIdx.x / tiles, t0 = blockIdx.x % tiles * kTile;
  const int nt = (int)(p.N - t0 < kTile ? p.N - t0 : kTile);
  stage_angles(p, b, t0, nt, cs);
  __syncthreads();
  const int D = p.D, half = D / 2;  // pairs, then the rest of the head two by two
  const int64_t heads = p.H + 2 * p.Hk;
  for (int64_t i = threadIdx.x; i < nt * heads * half; i += kThreads) {
    const int q = (int)(i % half);
    const int64_t h = i / half % heads;
    const int t = (int)(i / (half * heads));
    const int64_t n = t0 + t;
    int2 e = make_int2(2 * q, 2 * q + 1);
    float2 turn = make_float2(1.0f, 0.0f);
    if (h < p.H + p.Hk && q < p.pairs) {
      e = pair_at(p, q);
      turn = cs[t * p.pairs + q];
    }
    const int64_t fused = ((b * p.N + n) * heads + h) * D;
    T *head;
    int64_t step = 1;
    if (h < p.H) {
      head = static_cast<T *>(p.q) + ((b * p.H + h) * p.N + n) * D;
    } else if (h < p.H + p.Hk) {
      head = static_cast<T *>(p.k) + ((b * p.Hk + h - p.H) * p.N + n) * D;
    } else if (p.v_transposed) {
      head = static_cast<T *>(p.v) + (b * p.Hk + h - p.H - p.Hk) * D * p.N + n;
      step = p.N;
    } else {
      head = static_cast<T *>(p.v) + ((b * p.Hk + h - p.H - p.Hk) * p.N + n) * D;
    }
    T *fu = static_cast<T *>(p.qkv) + fused + e.x, *fv = static_cast<T *>(p.qkv) + fused + e.y;
    T *hu = head + e.x * step, *hv = head + e.y * step;
    if (h >= p.H + p.Hk || q >= p.pairs) {  // copied bit for bit
      if (kBackward) {
        *fu = *hu;
        *fv = *hv;
      } else {
        *hu = *fu;
        *hv = *fv;
      }
      continue;
    }
    const float u = to_f32(kBackward ? *hu : *fu), v = to_f32(kBackward ? *hv : *fv);
    const T ru = from_f32<T>(__fmaf_rn(u, turn.x, -v * turn.y));
    const T rv = from_f32<T>(__fmaf_rn(v, turn.x, u * turn.y));
    if (kBackward) {
      *fu = ru;
      *fv = rv;
    } else {
      *hu = ru;
      *hv = rv;
    }
  }
}

template <typename T>
cudaError_t launch(const RotaryParams &p, cudaStream_t s) {
  const int64_t blocks = p.B * ((p.N + kTile - 1) / kTile);
  const size_t smem = (size_t)kTile * p.pairs * sizeof(float2);  // <= 32 KB (D <= 256)
  if (p.inverse)
    rotary_kernel<T, true><<<(unsigned)blocks, kThreads, smem, s>>>(p);
  else
    rotary_kernel<T, false><<<(unsigned)blocks, kThreads, smem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams &p, int dtype, cudaStream_t s) {
  if (dtype == SCMP_F32) return launch<float>(p, s);
  if (dtype == SCMP_BF16) return launch<__nv_bfloat16>(p, s);
  return launch<__half>(p, s);
}

}  // namespace scmp
