// The fused qkv projection output split into q, k and v with q and k turned by
// multi-axis rotary positions, and its gradient.
//   pair (u, v) of axis a, frequency i, at coordinate c:
//     u' = u cos t - v sin t,  v' = v cos t + u sin t,  t = c scale_a base^(-2 i / d_a)
// cos and sin come from a table per axis (rows = coordinates), built in 64 bits
// where far coordinates need them; the backward pass turns by -t.
//
// A thread owns a piece of a token's head (16 bytes, fewer where sizes or pointers
// ask for it) and walks the heads: its cos and sin stay in
// registers, every access of a warp covers whole head rows, and a few heads are
// in flight at a time.  v with its dimensions and tokens exchanged goes through
// a shared-memory tile in blocks of its own, in the same launch.  HBM-bound: 64
// images of 16 heads of 64 in 38 us (bf16, 5.3 TB/s) and 67 us (fp32, 6.0 TB/s).
#include "mx_common.cuh"
#include "rotary.cuh"
#include "rotary_device.cuh"

namespace scmp {
namespace {

constexpr int kAtOnce = 4;  // heads in flight per thread

// x turned: x cos + partner (-+ sin); words that stay are x's bits.
template <typename T, int V, bool kInterleaved>
__device__ __forceinline__ Piece<T, V> turned(const Piece<T, V> &x, const Piece<T, V> &o,
                                              const float (&c)[V], const float (&s)[V],
                                              uint32_t mask) {
  Piece<T, V> r;
  if constexpr (V == 1) {
    r.u[0] = mask ? from_f32<T>(__fmaf_rn(to_f32(x.u[0]), c[0], to_f32(o.u[0]) * s[0])) : x.u[0];
  } else {
    float v[V], w[V];
    x.get(v);
    if (kInterleaved) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = v[i ^ 1];
    } else {
      o.get(w);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = __fmaf_rn(v[i], c[i], w[i] * s[i]);
    constexpr int kPer = 4 / (int)sizeof(T);  // elements per word: a pair's, or one
#pragma unroll
    for (int i = 0; i < V / kPer; ++i)
      r.u[i] = (mask >> (i * kPer)) & 1 ? Piece<T, V>::word(v, i) : x.u[i];
  }
  return r;
}

template <typename T, int V, bool kInterleaved, bool kBackward>
__device__ __forceinline__ void turn_heads(const RotaryParams &p, uint32_t block) {
  const int per = p.D / V;  // pieces of a head row
  const uint32_t id = (block / p.splits) * kThreads + threadIdx.x;  // of B N per pieces
  const uint32_t tok = p.per.quotient(id);
  if (tok >= (uint32_t)(p.B * p.N)) return;
  const uint32_t b = p.tokens.quotient(tok), n = tok - b * (uint32_t)p.N;
  const int e0 = (int)(id - tok * per) * V;
  const int heads = (int)(p.H + 2 * p.Hk), turning = (int)(p.H + p.Hk);
  const int all = p.v_transposed ? turning : heads;
  const int first = (int)(block % p.splits) * p.heads_per;
  const int last = first + p.heads_per < all ? first + p.heads_per : all;

  float c[V], s[V];
  int partner;
  const uint32_t mask = angles_of<V, kInterleaved, kBackward>(
      p, p.pos_batched ? tok : n, e0, c, s, partner);
  const bool fetch = (!kInterleaved || V == 1) && mask != 0;

  T *const fused = static_cast<T *>(p.qkv) + (int64_t)tok * heads * p.D;
  for (int h0 = first; h0 < last; h0 += kAtOnce) {
    Piece<T, V> x[kAtOnce], o[kAtOnce];
    T *to[kAtOnce], *from[kAtOnce];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      const int h = h0 + q < last ? h0 + q : last - 1;
      T *base;
      int hh = h;
      int64_t count = p.H;
      if (h < p.H) {
        base = static_cast<T *>(p.q);
      } else {
        base = static_cast<T *>(h < turning ? p.k : p.v);
        hh = h - (int)(h < turning ? p.H : turning);
        count = p.Hk;
      }
      T *const head = base + (((int64_t)b * count + hh) * p.N + n) * p.D;
      T *const row = fused + (int64_t)h * p.D;
      from[q] = kBackward ? head : row;
      to[q] = kBackward ? row : head;
      x[q].load(from[q] + e0);
      if (fetch && h < turning) o[q].load(from[q] + partner);
    }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      if (h0 + q >= last) break;
      if (mask != 0 && h0 + q < turning)
        turned<T, V, kInterleaved>(x[q], o[q], c, s, mask).store(to[q] + e0);
      else
        x[q].store(to[q] + e0);
    }
  }
}

template <typename T, int V, bool kInterleaved, bool kBackward>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  if (blockIdx.x < p.turn_blocks)
    turn_heads<T, V, kInterleaved, kBackward>(p, blockIdx.x);
  else
    transpose_tile<T, V, kBackward>(p, blockIdx.x - p.turn_blocks, reinterpret_cast<T *>(smem));
}

template <typename T, int V, bool kInterleaved>
cudaError_t launch_v(RotaryParams p, cudaStream_t s) {
  p.per = FastDiv((uint32_t)(p.D / V));
  p.tokens = FastDiv((uint32_t)p.N);
  const int all = (int)(p.H + p.Hk + (p.v_transposed ? 0 : p.Hk));
  const int64_t token_blocks = (p.B * p.N * (p.D / V) + kThreads - 1) / kThreads;
  // as many heads per thread as leave six blocks for each of the 148 SMs
  const int64_t fit = all * token_blocks / (148 * 6);
  p.heads_per = (int)(fit < 1 ? 1 : fit > all ? all : fit);
  p.splits = (uint32_t)((all + p.heads_per - 1) / p.heads_per);
  const int64_t turn = token_blocks * p.splits;
  const int64_t tiles = p.v_transposed ? p.B * p.Hk * ((p.N + kTile - 1) / kTile) : 0;
  if (turn + tiles > INT32_MAX) return cudaErrorInvalidConfiguration;
  p.turn_blocks = (uint32_t)turn;
  const size_t smem = p.v_transposed ? (size_t)(kTile + 2) * p.D * sizeof(T) : 0;  // <= 66 KB
  auto kern = p.inverse ? rotary_kernel<T, V, kInterleaved, true>
                        : rotary_kernel<T, V, kInterleaved, false>;
  if (smem > 48 * 1024) {
    // (always the most that this kernel uses: calls at the same time agree on it)
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (kTile + 2) * 256 * (int)sizeof(T));
    if (e != cudaSuccess) return e;
  }
  kern<<<(unsigned)(turn + tiles), kThreads, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, bool kInterleaved>
cudaError_t launch_order(const RotaryParams &p, cudaStream_t s) {
  constexpr int V = kVec16<T>;
  if (pieces<T, V>(p)) return launch_v<T, V, kInterleaved>(p, s);
  if (pieces<T, V / 2>(p)) return launch_v<T, V / 2, kInterleaved>(p, s);
  if constexpr (sizeof(T) == 2)
    if (pieces<T, V / 4>(p)) return launch_v<T, V / 4, kInterleaved>(p, s);
  return launch_v<T, 1, kInterleaved>(p, s);
}
template <typename T> cudaError_t launch(const RotaryParams &p, cudaStream_t s) {
  return p.interleaved ? launch_order<T, true>(p, s) : launch_order<T, false>(p, s);
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams &p, int dtype, cudaStream_t s) {
  if (dtype == SCMP_F32) return launch<float>(p, s);
  if (dtype == SCMP_BF16) return launch<__nv_bfloat16>(p, s);
  return launch<__half>(p, s);
}

}  // namespace scmp
