// Gated residual add with the norms around it, in one pass over the rows, and
// its gradients:
//   z = y, or N(y) pw + pb (a norm behind the branch)
//   r = x + z gamma gate          rounded to x's type
//   h = N(r) w + b                the norm in front of the next branch
// N(v) = (v - mean) / sqrt(var + eps), or v / sqrt(mean v^2 + eps).  A row stays
// in registers from its loads to its stores; statistics are fp32, the variance
// a second pass over the registers.
#include "norm.cuh"

#include "f32x2.cuh"
#include "mx_common.cuh"

namespace scmp {
namespace {

// A row is dealt to G warps: chunk j (of NV, each V consecutive columns per lane)
// of warp w starts at column ((j G + w) 32 + lane) V.  Single elements: at (w NV +
// j) 32 + lane, so that a lane's columns are a constant distance apart (with the
// order above, computing their addresses took rows of 1001 elements to 132 us
// forward and 334 backward, at 16448 rows of bf16).
template <int V, int NV> __device__ __forceinline__ int col_of(int j, int G, int w, int lane) {
  return V == 1 ? (w * NV + j) * 32 + lane : ((j * G + w) * 32 + lane) * V;
}

// V consecutive elements, as loaded: 16-byte pieces, or one element (V = 1).
template <typename T, int V> struct Pack {
  static constexpr int kN = V * (int)sizeof(T) / 16;
  uint4 u[kN];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kN; ++i) u[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < kN; ++i) u[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
  }
  __device__ __forceinline__ void get(float *v) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) unpack16<T>(u[i], v + i * kVec16<T>);
  }
};
template <typename T> struct Pack<T, 1> {
  T u;
  __device__ __forceinline__ void zero() { u = from_f32<T>(0.0f); }
  __device__ __forceinline__ void load(const T *p) { u = *p; }
  __device__ __forceinline__ void get(float *v) const { v[0] = to_f32(u); }
};
template <typename T, int V> __device__ __forceinline__ void load_v(const T *p, float *v) {
  Pack<T, V> q;
  q.load(p);
  q.get(v);
}
template <typename T, int V> __device__ __forceinline__ void store_v(T *p, const float *v) {
  if (V == 1) {
    *p = from_f32<T>(v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += kVec16<T>)
      *reinterpret_cast<uint4 *>(p + i) = pack16<T>(v + i);
  }
}
// 16-byte pieces stored, and v becomes the rounded values.
template <typename T, int V> __device__ __forceinline__ void store_rounded(T *p, float *v) {
#pragma unroll
  for (int i = 0; i < V; i += kVec16<T>) {
    const uint4 u = pack16<T>(v + i);
    *reinterpret_cast<uint4 *>(p + i) = u;
    unpack16<T>(u, v + i);
  }
}

// The E values of a lane, chunk j's V from element j V on, as pairs.
template <int E> struct Values {
  float2 p[E / 2];
  __device__ __forceinline__ float *at(int e) { return reinterpret_cast<float *>(p) + e; }
};

constexpr int kMaxWarps = 16;

// Sums over the G warps of a row slot, which meet at a barrier of their own.
// Two buffers in turn: a warp writes one again only after the barrier that
// follows every read of it.
struct RowSum {
  float2 *buf;  // this slot's warps in [2][kMaxWarps], an even number (the last may be 0)
  int G, w, barrier, turn;
  __device__ RowSum(float2 *all, int G_, int slot, int w_)
      : buf(all + slot * ((G_ + 1) & ~1)), G(G_), w(w_), barrier(1 + slot), turn(0) {
    if ((G & 1) && w == 0 && (threadIdx.x & 31) == 0)
      buf[G] = buf[kMaxWarps + G] = make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ float2 meet() {
    const float4 *b = reinterpret_cast<const float4 *>(buf + turn * kMaxWarps);
    turn ^= 1;
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(G * 32) : "memory");
    float2 v = make_float2(0.f, 0.f);
    const auto add = [&](int i) {
      if (2 * i >= G) return;
      const float4 f = b[i];
      v.x += f.x;
      v.y += f.y;
      v.x += f.z;
      v.y += f.w;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) add(i);
    if (G > 8) {
#pragma unroll
      for (int i = 4; i < kMaxWarps / 2; ++i) add(i);
    }
    return v;
  }
  // (half the lanes go on with x, the others with y)
  __device__ __forceinline__ float2 operator()(float2 v) {
    const bool hi = threadIdx.x & 16;
    float a = hi ? v.y : v.x;
    a += __shfl_xor_sync(~0u, hi ? v.x : v.y, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(~0u, a, o);
    if (G == 1) return make_float2(__shfl_sync(~0u, a, 0), __shfl_sync(~0u, a, 16));
    if ((threadIdx.x & 15) == 0)
      reinterpret_cast<float *>(buf + turn * kMaxWarps + w)[hi ? 1 : 0] = a;
    return meet();
  }
  __device__ __forceinline__ float operator()(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (G == 1) return v;
    if ((threadIdx.x & 31) == 0) buf[turn * kMaxWarps + w] = make_float2(v, 0.f);
    return meet().x;
  }
};

// v (0 past the row, where in(j) is false) -> N(v) and its statistics.
template <int V, int E, typename In>
__device__ __forceinline__ float2 normalise(Values<E> &v, const In &in, RowSum &sum, float inv_c,
                                            float eps, bool rms) {
  float mean = 0.f;
  if (!rms) {
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) s = add2(s, v.p[i]);
    mean = sum(s.x + s.y) * inv_c;
#pragma unroll
    for (int i = 0; i < E / 2; ++i)  // (what lies past the row stays 0)
      v.p[i] = add2(v.p[i], make_float2(in(2 * i / V) ? -mean : 0.f,
                                        in((2 * i + 1) / V) ? -mean : 0.f));
  }
  float2 q = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < E / 2; ++i) q = fma2(v.p[i], v.p[i], q);
  const float rstd = 1.0f / sqrtf(__fmaf_rn(sum(q.x + q.y), inv_c, eps));
#pragma unroll
  for (int i = 0; i < E / 2; ++i) v.p[i] = mul2(v.p[i], both(rstd));
  return make_float2(mean, rstd);
}

// V values of a block of the 4-bit formats per lane: their codes and, from the
// block's largest magnitude over the lanes that hold it, the row's scale words.
template <int kFmt, int V>
__device__ __forceinline__ void store_mx(const NormParams &p, const float *v, int64_t row, int col,
                                         int lane) {
  constexpr int kBlock = kFmt == SCMP_MXFP4 ? 32 : 16;
  constexpr int kLanes = kBlock / V;
  float v8[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v8[i] = i < V ? v[i] : 0.f;
  uint32_t amax = max_bits<V>(v), codes;
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) amax = max(amax, __shfl_xor_sync(~0u, amax, o));
  const uint32_t scale = mx_encode8<kFmt, false>(v8, amax, 1.0f, &codes);
  if (row < p.rows && col < p.kp) {
    uint8_t *d = p.mx_data + row * (p.kp >> 1) + (col >> 1);
    if (V == 8)
      *reinterpret_cast<uint32_t *>(d) = codes;
    else
      *reinterpret_cast<uint16_t *>(d) = (uint16_t)codes;
  }
  const int blk = col / kBlock;
  if ((lane & (kLanes - 1)) == 0 && (blk >> 2) < p.groups)
    p.mx_scales[mx_scale_word(row, blk >> 2, p.groups) + (blk & 3)] = (uint8_t)scale;
}

// E elements per lane, by the shape (rows x columns, bf16 unless fp32, us):
//   E = 8   one row per slot, up to 2048 columns: a short chain per row and 48
//           warps an SM.  Few rows (257 x 1024: 3.2, E = 16 3.5), fp32 rows that
//           fill blocks of eight warps (16448 x 1024: 49.6 = a copy's rate, E = 16
//           57.9; 8200 x 2048: 50.3, 54.2), rows of one warp (16448 x 200: 9.4,
//           E = 16 10.7)
//   E = 16  slots walk rows, and once a row's x and y are used the next one is on
//           its way into their registers.  Many rows (16448 x 1024: 27.1, E = 8
//           42.1; fp32 16400 x 1408: 69.9, E = 8 79.4, with a post norm 85.6, 111)
//   E = 32  the same for rows of over 4096 columns
// Rows not in 16-byte pieces go one element at a time: E = 8 up to 2048 columns
// (16448 x 1001: 67 us, E = 16 71; fp32 69, 99), E = 16 up to 4096, two blocks an
// SM rather than three, which spill (6400 x 2501: 73, 82).
// 16-bit rows are bound by instructions: two fp32 operations per instruction, the
// gate's row by a multiplication and sums over lanes in half the shuffles took
// 16400 x 1408 with gates and a post norm from 57 to 46 us.
template <typename T, typename P, int V, int E>
__global__ void __launch_bounds__(256, E == 16 ? (V == 1 ? 2 : 3) : 1)
    residual_norm_kernel(const __grid_constant__ NormParams p) {
  constexpr bool kWalk = E > 8;
  constexpr int NV = E / V;
  __shared__ __align__(16) float2 buf[2 * kMaxWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.warps_per_row, slot = warp / G, w = warp - slot * G;
  const int slots = blockDim.x / (32 * G);
  RowSum sum(buf, G, slot, w);
  const int C = p.C;
  const float inv_c = 1.0f / (float)C;
  const auto in_row = [&](int j) { return col_of<V, NV>(j, G, w, lane) < C; };

  Pack<T, V> x[NV], y[NV];
  const auto load = [&](int64_t row) {
    const bool live = row < p.rows;
    const int64_t at = row * C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x[j].zero();
      y[j].zero();
      if (!live || !in_row(j)) continue;
      const int c = col_of<V, NV>(j, G, w, lane);
      x[j].load(static_cast<const T *>(p.x) + at + c);
      if (p.y) y[j].load(static_cast<const T *>(p.y) + at + c);
    }
  };
  // (rows past the last one, up to a multiple of 128, exist for 4-bit scales)
  const int64_t stride = (int64_t)gridDim.x * slots;
  int64_t row = (int64_t)blockIdx.x * slots + slot;
  load(row);
  for (; row < p.row_end; row = kWalk ? row + stride : p.row_end) {
    const bool live = row < p.rows;
    const auto in = [&](int j) { return live && in_row(j); };
    const int64_t at = row * C;
    Values<E> r;
    if (p.y) {
#pragma unroll
      for (int j = 0; j < NV; ++j) y[j].get(r.at(j * V));
      if (p.post_weight) {
        const float2 st = normalise<V, E>(r, in, sum, inv_c, p.eps, p.rms);
        if (p.stats && live && w == 0 && lane == 0) p.stats[p.rows + row] = st;
      }
      const int64_t gate_at = p.gate && live ? (int64_t)p.per_gate.quotient((uint32_t)row) * C : 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        // (single elements past the row go along, reading its last parameters,
        // rather than branch)
        const bool ok = in(j);
        const int c0 = col_of<V, NV>(j, G, w, lane), c = V > 1 || c0 < C ? c0 : C - 1;
        float *const rj = r.at(j * V);
        if (V > 1 && !ok) {
#pragma unroll
          for (int i = 0; i < V; ++i) rj[i] = 0.f;
          continue;
        }
        constexpr int N2 = V > 1 ? V / 2 : 1;
        float2 z[N2], f[N2], g[N2];
        const auto load2 = [&](const void *src, int64_t at, float2 *to) {
          if (V == 1) to[0].y = 0.f;
          load_v<P, V>(static_cast<const P *>(src) + at, &to[0].x);
        };
#pragma unroll
        for (int i = 0; i < N2; ++i)
          z[i] = make_float2(rj[2 * i], V > 1 ? rj[2 * i + (V > 1)] : 0.f);
        if (p.post_weight) {
          load2(p.post_weight, c, f);
          if (p.post_bias) {
            load2(p.post_bias, c, g);
#pragma unroll
            for (int i = 0; i < N2; ++i) z[i] = add2(mul2(z[i], f[i]), g[i]);
          } else {
#pragma unroll
            for (int i = 0; i < N2; ++i) z[i] = mul2(z[i], f[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < N2; ++i) f[i] = both(1.0f);
        if (p.gamma) load2(p.gamma, c, f);
        if (p.gate) {
          load2(p.gate, gate_at + c, g);
#pragma unroll
          for (int i = 0; i < N2; ++i) f[i] = mul2(f[i], g[i]);
        }
        x[j].get(&g[0].x);
        if (V == 1) g[0].y = 0.f;
#pragma unroll
        for (int i = 0; i < N2; ++i) {
          z[i] = fma2(z[i], f[i], g[i]);
          rj[2 * i] = z[i].x;
          if (V > 1) rj[2 * i + (V > 1)] = z[i].y;
        }
        // r is rounded to its type once, and the norm sees the rounded value:
        // the one that the next block and the backward pass read
        if (V == 1) {
          const T t = from_f32<T>(rj[0]);
          if (ok) static_cast<T *>(p.r)[at + c] = t;
          rj[0] = ok ? to_f32(t) : 0.f;
        } else {
          store_rounded<T, V>(static_cast<T *>(p.r) + at + c, rj);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) x[j].get(r.at(j * V));
    }
    if (kWalk) load(row + stride);
    const float2 st = normalise<V, E>(r, in, sum, inv_c, p.eps, p.rms);
    if (p.stats && live && w == 0 && lane == 0) p.stats[row] = st;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool ok = in(j);
      const int c0 = col_of<V, NV>(j, G, w, lane), c = V > 1 || c0 < C ? c0 : C - 1;
      float *const rj = r.at(j * V);
      if (V == 1 || ok) {
        constexpr int N2 = V > 1 ? V / 2 : 1;
        float2 z[N2], f[N2], g[N2];
        const auto load2 = [&](const void *src, float2 *to) {
          if (V == 1) to[0].y = 0.f;
          load_v<P, V>(static_cast<const P *>(src) + c, &to[0].x);
        };
#pragma unroll
        for (int i = 0; i < N2; ++i)
          z[i] = make_float2(rj[2 * i], V > 1 ? rj[2 * i + (V > 1)] : 0.f);
        load2(p.weight, f);
        if (p.bias) {
          load2(p.bias, g);
#pragma unroll
          for (int i = 0; i < N2; ++i) z[i] = fma2(z[i], f[i], g[i]);
        } else {
#pragma unroll
          for (int i = 0; i < N2; ++i) z[i] = mul2(z[i], f[i]);
        }
#pragma unroll
        for (int i = 0; i < N2; ++i) {
          rj[2 * i] = z[i].x;
          if (V > 1) rj[2 * i + (V > 1)] = z[i].y;
        }
        if (p.h && ok) {
          if (p.h_f32)
            store_v<float, V>(static_cast<float *>(p.h) + at + c, rj);
          else
            store_v<T, V>(static_cast<T *>(p.h) + at + c, rj);
        }
      } else {  // (0 times a deviation's reciprocal that is infinite)
#pragma unroll
        for (int i = 0; i < V; ++i) rj[i] = 0.f;
      }
      if (V > 1 && p.mx_data) {
        if (p.fmt == SCMP_MXFP4)
          store_mx<SCMP_MXFP4, V>(p, rj, row, c, lane);
        else
          store_mx<SCMP_NVFP4, V>(p, rj, row, c, lane);
      }
    }
  }
}

// ---------------------------------------------------------------- backward
// Rows of one gate group (all rows without a gate) are dealt to row slots of G
// warps; a block holds a few slots of one group.  Column sums stay in registers
// over a slot's rows, are added over the block's slots in shared memory in a
// fixed order and written as partials [group][block][part][C]; a second kernel
// adds those in order, so the result does not depend on timing.
//   parts: 0 sum dh n   1 sum dh   2 sum g z (no post norm) or sum g m   3 sum g
// E = 8 elements per lane for rows of up to 2048, else 16.
//
// A slot's next rows are on their way into a ring of stages in shared memory,
// each thread copying what it will read itself (no barrier), which leaves the
// registers to the sums; with a post norm the parameters stay there too.  bf16
// 16448 x 1024: 39 us (5.2 TB/s), in registers one row ahead 45; fp32 73 (5.5);
// 16400 x 1408 with gates and a post norm bf16 76 us, 102 with registers and
// single operations, when instructions bounded it; now 52 % of cycles issue and the
// two meetings of a row's warps are left; fp32 105 (5.3 TB/s), 201.  Rows not in
// 16-byte pieces, and fp32 rows of over 4096 columns, whose ring would not fit, load
// as they go.
template <typename T, int V, int E, int kThreads> struct BwdCfg {
  static constexpr int kPieces = E * (int)sizeof(T) / 16;  // 16-byte pieces per array and lane
  static constexpr int kStages = V == 1 ? 0
                                 : E == 8 || kThreads == 256 ? (sizeof(T) == 2 ? 4 : 3)
                                                             : (sizeof(T) == 2 ? 3 : 0);
  // bytes per thread and stage; each warp's two statistics behind them
  static constexpr int kStageBytes = 4 * kPieces * 16;
};
__device__ __forceinline__ void copy_async16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_async8(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src)
               : "memory");
}

template <typename T, typename P, int V, int E, bool kPost, int kThreads>
__global__ void __launch_bounds__(kThreads, E == 8 ? 2 : 1)
    residual_norm_bwd_kernel(const __grid_constant__ NormBwdParams p) {
  using Cfg = BwdCfg<T, V, E, kThreads>;
  constexpr int NV = E / V;
  constexpr int kParts = kPost ? 4 : 3;
  constexpr int kStages = Cfg::kStages, kPieces = Cfg::kPieces;
  constexpr bool kHeld = !(kPost && E == 8 && V > 1);  // parameters in registers, else in shared memory
  __shared__ __align__(16) float2 buf[2 * kMaxWarps];
  __shared__ float2 stat_ring[kStages > 0 ? kStages : 1][kMaxWarps][2];
  extern __shared__ __align__(16) unsigned char smem[];
  float *const part_smem = reinterpret_cast<float *>(smem);  // [C], once the rows are done
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.warps_per_row, slot = warp / G, w = warp - slot * G;
  const int slots = blockDim.x / (32 * G);
  RowSum sum(buf, G, slot, w);
  const int C = p.C;
  const float inv_c = 1.0f / (float)C;
  const int64_t group = blockIdx.x / p.blocks_per_group;
  const int64_t stride = p.blocks_per_group * slots;
  const int64_t row0 = group * p.rows_per_group;

  // [stage][array][piece][thread], then the parameters in shared memory
  uint4 *const ring = reinterpret_cast<uint4 *>(smem) + threadIdx.x;
  const int per_array = kPieces * (int)blockDim.x, per_stage = 4 * per_array;
  const T *const array[4] = {static_cast<const T *>(p.r), static_cast<const T *>(p.dh),
                             static_cast<const T *>(p.dr), static_cast<const T *>(p.y)};
  const auto fetch = [&](int64_t i_row, int stage) {
    if (i_row < p.rows_per_group) {
      const int64_t row = row0 + i_row;
      if (lane == 0) {
        copy_async8(&stat_ring[stage][warp][0], p.stats + row);
        if (kPost) copy_async8(&stat_ring[stage][warp][1], p.stats + p.rows + row);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = col_of<V, NV>(j, G, w, lane);
        if (c >= C) continue;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          if (!array[a]) continue;
          const T *src = array[a] + row * C + c;
          uint4 *dst = ring + stage * per_stage + a * per_array + j * (kPieces / NV) * blockDim.x;
#pragma unroll
          for (int k = 0; k < kPieces / NV; ++k)
            copy_async16(dst + k * blockDim.x, src + k * kVec16<T>);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // V elements of an array's chunk j in this stage (or straight from memory)
  const auto get = [&](int a, int j, int stage, int64_t at, float *v) {
    if constexpr (kStages > 0) {
      const uint4 *src = ring + stage * per_stage + a * per_array + j * (kPieces / NV) * blockDim.x;
#pragma unroll
      for (int k = 0; k < kPieces / NV; ++k) unpack16<T>(src[k * blockDim.x], v + k * kVec16<T>);
    } else {
      // (the raw element is what the predicate guards: no branch per element)
      const int c = col_of<V, NV>(j, G, w, lane);
      Pack<T, V> q;
      q.zero();
      if (c < C && array[a]) q.load(array[a] + at + c);
      q.get(v);
    }
  };
  if constexpr (kStages > 0) {
    // what no copy writes (columns past the row, arrays that are not there) is 0
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        if (col_of<V, NV>(j, G, w, lane) >= C || !array[a])
          for (int s = 0; s < kStages; ++s)
            for (int k = 0; k < kPieces / NV; ++k)
              ring[s * per_stage + a * per_array + (j * (kPieces / NV) + k) * blockDim.x] =
                  make_uint4(0, 0, 0, 0);
  }
  int64_t i_row = (blockIdx.x % p.blocks_per_group) * slots + slot;
#pragma unroll
  for (int s = 0; s + 1 < kStages; ++s) fetch(i_row + s * stride, s);

  // the parameters of this lane's columns stay the same over the rows: weight
  // and gamma gate (times post_weight)
  float wt[kHeld ? NV : 1][V], sc[kHeld ? NV : 1][V];
  float4 *const held = reinterpret_cast<float4 *>(smem) + kStages * 4 * kPieces * blockDim.x +
                       w * (E / 4) * 32 + lane;
  const int plane = G * (E / 4) * 32;
  if (kHeld || slot == 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col_of<V, NV>(j, G, w, lane), k = kHeld ? j : 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        wt[k][i] = 0.f;
        sc[k][i] = kPost ? 0.f : 1.f;
      }
      if (c < C) {
        float f[V];
        load_v<P, V>(static_cast<const P *>(p.weight) + c, wt[k]);
        if (kPost) load_v<P, V>(static_cast<const P *>(p.post_weight) + c, sc[k]);
        if (p.gamma) {
          load_v<P, V>(static_cast<const P *>(p.gamma) + c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) sc[k][i] *= f[i];
        }
        if (p.gate) {
          load_v<P, V>(static_cast<const P *>(p.gate) + group * C + c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) sc[k][i] *= f[i];
        }
      }
      if constexpr (!kHeld) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          float4 *const to = held + (j * V + i) / 4 * 32;
          to[0] = make_float4(wt[0][i], wt[0][i + 1], wt[0][i + 2], wt[0][i + 3]);
          to[plane] = make_float4(sc[0][i], sc[0][i + 1], sc[0][i + 2], sc[0][i + 3]);
        }
      }
    }
  }
  if (!kHeld) __syncthreads();
  const auto param = [&](int which, int j, float *v) {
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = which ? sc[j][i] : wt[j][i];
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 f = held[which * plane + (j * V + i) / 4 * 32];
        v[i] = f.x;
        v[i + 1] = f.y;
        v[i + 2] = f.z;
        v[i + 3] = f.w;
      }
    }
  };
  Values<E> acc[kParts];
#pragma unroll
  for (int k = 0; k < kParts; ++k)
#pragma unroll
    for (int i = 0; i < E / 2; ++i) acc[k].p[i] = make_float2(0.f, 0.f);

  int stage = 0;
  for (; i_row < p.rows_per_group; i_row += stride) {
    const int64_t row = row0 + i_row, at = row * C;
    float2 st, st_y = make_float2(0.f, 0.f);
    if constexpr (kStages > 0) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages > 1 ? kStages - 2 : 0) : "memory");
      __syncwarp();  // lane 0 fetched the statistics
      st = stat_ring[stage][warp][0];
      if (kPost) st_y = stat_ring[stage][warp][1];
      __syncwarp();
      // into the stage that the row before this one was read from
      fetch(i_row + (kStages - 1) * stride, stage == 0 ? kStages - 1 : stage - 1);
    } else {
      st = p.stats[row];
      if (kPost) st_y = p.stats[p.rows + row];
    }
    const auto in = [&](int j) { return col_of<V, NV>(j, G, w, lane) < C; };
    Values<E> n, dn, f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      get(0, j, stage, at, n.at(j * V));
      get(1, j, stage, at, dn.at(j * V));
      param(0, j, f.at(j * V));
    }
    float2 s = make_float2(0.f, 0.f), t = s;  // pairs of sums of dn and of dn n
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 mean = make_float2(in(2 * i / V) ? -st.x : 0.f, in((2 * i + 1) / V) ? -st.x : 0.f);
      n.p[i] = mul2(add2(n.p[i], mean), both(st.y));
      acc[0].p[i] = fma2(dn.p[i], n.p[i], acc[0].p[i]);
      acc[1].p[i] = add2(acc[1].p[i], dn.p[i]);
      dn.p[i] = mul2(dn.p[i], f.p[i]);
      s = add2(s, dn.p[i]);
      t = fma2(dn.p[i], n.p[i], t);
    }
    s = sum(make_float2(s.x + s.y, t.x + t.y));
    const float2 mean_dn = both(p.rms ? 0.f : -s.x * inv_c), mean_dnn = both(-s.y * inv_c);
    Values<E> g, y;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      get(2, j, stage, at, g.at(j * V));
      get(3, j, stage, at, y.at(j * V));
      param(1, j, f.at(j * V));
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i)
      g.p[i] = fma2(both(st.y), fma2(n.p[i], mean_dnn, add2(dn.p[i], mean_dn)), g.p[i]);
    const auto store = [&](void *to, Values<E> &v) {
      if (!to) return;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (in(j)) store_v<T, V>(static_cast<T *>(to) + at + col_of<V, NV>(j, G, w, lane), v.at(j * V));
    };
    store(p.dx, g);
    if (kPost) {
      s = t = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 mean =
            make_float2(in(2 * i / V) ? -st_y.x : 0.f, in((2 * i + 1) / V) ? -st_y.x : 0.f);
        y.p[i] = mul2(add2(y.p[i], mean), both(st_y.y));
        acc[2].p[i] = fma2(g.p[i], y.p[i], acc[2].p[i]);
        acc[kParts - 1].p[i] = add2(acc[kParts - 1].p[i], g.p[i]);
        g.p[i] = mul2(g.p[i], f.p[i]);
        s = add2(s, g.p[i]);
        t = fma2(g.p[i], y.p[i], t);
      }
      s = sum(make_float2(s.x + s.y, t.x + t.y));
      const float2 mean_dm = both(p.rms ? 0.f : -s.x * inv_c), mean_dmm = both(-s.y * inv_c);
#pragma unroll
      for (int i = 0; i < E / 2; ++i)
        g.p[i] = mul2(both(st_y.y), fma2(y.p[i], mean_dmm, add2(g.p[i], mean_dm)));
    } else {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        acc[2].p[i] = fma2(g.p[i], y.p[i], acc[2].p[i]);
        g.p[i] = mul2(g.p[i], f.p[i]);
      }
    }
    store(p.dy, g);
    if (kStages > 0) stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  if (kStages > 0) asm volatile("cp.async.wait_all;" ::: "memory");
  if (!p.part) return;
  if (kStages > 0) __syncthreads();  // the ring's place is taken by the sums
  float *out = p.part + (int64_t)blockIdx.x * 4 * C;
#pragma unroll
  for (int k = 0; k < kParts; ++k) {
    for (int q = slots - 1; q > 0; --q) {  // the slots add up, from the last to the first
      __syncthreads();
      if (slot == q) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int c = col_of<V, NV>(j, G, w, lane);
          if (c >= C) continue;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float v = acc[k].at(j * V)[i];
            if (q < slots - 1) v += part_smem[c + i];
            part_smem[c + i] = v;
          }
        }
      }
    }
    __syncthreads();
    if (slot == 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = col_of<V, NV>(j, G, w, lane);
        if (c >= C) continue;
#pragma unroll
        for (int i = 0; i < V; ++i)
          out[(int64_t)k * C + c + i] = acc[k].at(j * V)[i] + (slots > 1 ? part_smem[c + i] : 0.f);
      }
    }
  }
}

// The parameters' gradients of `groups` gate groups from the four column sums
// of each, columns of one thread.
template <typename P>
__device__ __forceinline__ void add_group(const NormBwdParams &p, int64_t group, int c,
                                          const float (&s)[4], float (&total)[5]) {
  const float gamma = p.gamma ? to_f32(static_cast<const P *>(p.gamma)[c]) : 1.0f;
  const float gate = p.gate ? to_f32(static_cast<const P *>(p.gate)[group * p.C + c]) : 1.0f;
  float gz = s[2];
  if (p.post_weight) {
    gz = s[2] * to_f32(static_cast<const P *>(p.post_weight)[c]);
    if (p.post_bias)
      gz = __fmaf_rn(s[3], to_f32(static_cast<const P *>(p.post_bias)[c]), gz);
  }
  total[0] += s[0];
  total[1] += s[1];
  total[2] = __fmaf_rn(gz, gate, total[2]);
  total[3] = __fmaf_rn(s[2], gamma * gate, total[3]);
  total[4] = __fmaf_rn(s[3], gamma * gate, total[4]);
  if (p.dgate) static_cast<P *>(p.dgate)[group * p.C + c] = from_f32<P>(gz * gamma);
}
template <typename P>
__device__ __forceinline__ void write_totals(const NormBwdParams &p, int c,
                                             const float (&total)[5]) {
  void *out[5] = {p.dweight, p.dbias, p.dgamma, p.dpost_weight, p.dpost_bias};
#pragma unroll
  for (int k = 0; k < 5; ++k)
    if (out[k]) static_cast<P *>(out[k])[c] = from_f32<P>(total[k]);
}

// The four sums of a group's partials, blocks first, first + step, ... of column c.
__device__ __forceinline__ void add_partials(const NormBwdParams &p, int64_t group, int first,
                                             int step, int c, int parts, float (&v)[4]) {
#pragma unroll 4
  for (int64_t b = first; b < p.blocks_per_group; b += step) {
    const float *src = p.part + (group * p.blocks_per_group + b) * 4 * p.C + c;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < parts) v[k] += __ldg(src + (int64_t)k * p.C);
  }
}

// One gate group: a block takes 8 columns, 32 or 128 threads per column share the
// partials.
template <typename P>
__global__ void __launch_bounds__(1024) norm_bwd_sum_kernel(
    const __grid_constant__ NormBwdParams p) {
  __shared__ float s[4][32][8];
  const int ci = threadIdx.x & 7, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (int)blockIdx.x * 8 + ci;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < p.C)
    add_partials(p, 0, threadIdx.x >> 3, blockDim.x >> 3, c, p.post_weight ? 4 : 3, v);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] += __shfl_xor_sync(~0u, v[k], 8);
    v[k] += __shfl_xor_sync(~0u, v[k], 16);
    if (lane < 8) s[k][warp][ci] = v[k];
  }
  __syncthreads();
  if (threadIdx.x >= 8 || c >= p.C) return;
  float one[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    one[k] = 0.f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) one[k] += s[k][i][ci];
  }
  float total[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  add_group<P>(p, 0, c, one, total);
  write_totals<P>(p, c, total);
}

// Several gate groups: a block takes 8 columns, of whose 64 or 128 threads each
// `p.share` (a power of two) share a group's partials; the groups' gradients are
// added over the threads.  Both sums are trees of a fixed shape.  (In two kernels,
// the groups' sums through memory: 64 groups of 1024 columns 19 us, now 7; 16384
// groups 313, now 180.)
template <typename P>
__global__ void __launch_bounds__(1024) norm_bwd_groups_kernel(
    const __grid_constant__ NormBwdParams p) {
  __shared__ float s[5][128][8];
  const int ci = threadIdx.x & 7, t = threadIdx.x >> 3;
  const int c = (int)blockIdx.x * 8 + ci, parts = p.post_weight ? 4 : 3;
  const int share = p.share, sub = t & (share - 1);
  float total[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  if (share == 1) {
    if (c < p.C) {
#pragma unroll 4
      for (int64_t g = t; g < p.groups; g += blockDim.x >> 3) {
        float one[4] = {0.f, 0.f, 0.f, 0.f};
        add_partials(p, g, 0, 1, c, parts, one);
        add_group<P>(p, g, c, one, total);
      }
    }
  } else {  // (share x groups threads or more)
    const int64_t g = t / share;
    const bool live = c < p.C && g < p.groups;
    float one[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) add_partials(p, g, sub, share, c, parts, one);
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k][t][ci] = one[k];
    for (int o = share >> 1; o > 0; o >>= 1) {
      __syncthreads();
      if (sub < o)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k][t][ci] += s[k][t + o][ci];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) one[k] = s[k][t][ci];
    if (live && sub == 0) add_group<P>(p, g, c, one, total);
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < 5; ++k) s[k][t][ci] = total[k];
  for (int o = (int)blockDim.x >> 4; o > 0; o >>= 1) {
    __syncthreads();
    if (t < o)
#pragma unroll
      for (int k = 0; k < 5; ++k) s[k][t][ci] += s[k][t + o][ci];
  }
  if (t > 0 || c >= p.C) return;
#pragma unroll
  for (int k = 0; k < 5; ++k) total[k] = s[k][0][ci];
  write_totals<P>(p, c, total);
}

// --------------------------------------------------------------- dispatch

// Backward: 8 elements per lane for rows of up to 2048.
bool short_rows(int64_t C) { return C <= 2048; }

template <typename T, typename P, int V, int E>
cudaError_t forward_e(NormParams p, cudaStream_t s) {
  const int G = (p.C + 32 * E - 1) / (32 * E), slots = 8 / G, threads = 32 * G * slots;
  p.warps_per_row = G;
  p.per_gate = FastDiv((uint32_t)p.rows_per_gate);
  p.row_end = p.mx_data ? (p.rows + 127) / 128 * 128 : p.rows;
  const int64_t blocks = (p.row_end + slots - 1) / slots;
  // walking slots: the blocks that 148 SMs hold at once
  const int64_t most = E == 8 ? blocks : 148 * ((E == 16 && V > 1 ? 768 : 512) / threads);
  residual_norm_kernel<T, P, V, E>
      <<<(unsigned)(blocks < most ? blocks : most), threads, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, typename P>
cudaError_t forward(const NormParams &p, bool vec, cudaStream_t s) {
  constexpr int V = kVec16<T>;
  if (!vec)
    return p.C <= 2048   ? forward_e<T, P, 1, 8>(p, s)
           : p.C <= 4096 ? forward_e<T, P, 1, 16>(p, s)
                         : forward_e<T, P, 1, 32>(p, s);
  const int G = (p.C + 255) / 256;  // warps per row at E = 8
  if (p.C <= 256 || (G <= 8 && ((sizeof(T) == 4 && 8 % G == 0) || p.rows <= 148 * 8)))
    return forward_e<T, P, V, 8>(p, s);
  return p.C <= 4096 ? forward_e<T, P, V, 16>(p, s) : forward_e<T, P, V, 32>(p, s);
}

template <typename T, typename P, int V, int E, int kThreads, bool kPost>
cudaError_t backward_post(const NormBwdParams &p, const NormBwdPlan &plan, cudaStream_t s) {
  using Cfg = BwdCfg<T, V, E, kThreads>;
  auto kern = residual_norm_bwd_kernel<T, P, V, E, kPost, kThreads>;
  const int threads = 32 * plan.warps_per_row * plan.slots;
  size_t smem = (size_t)Cfg::kStages * Cfg::kStageBytes * threads;
  if (kPost && E == 8 && V > 1) smem += (size_t)plan.warps_per_row * 32 * E * 2 * sizeof(float);
  const size_t sums = plan.slots > 1 ? (size_t)p.C * sizeof(float) : 0;
  if (smem < sums) smem = sums;
  if (smem > 44 * 1024) {  // (48 KB without asking, the kernel's own arrays included)
    // (always the most that this kernel uses: calls at the same time agree on it)
    constexpr size_t kMost = (size_t)Cfg::kStages * Cfg::kStageBytes * kThreads +
                             (kPost && E == 8 && V > 1 ? kThreads * E * 2 * sizeof(float) : 0);
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost);
    if (e != cudaSuccess) return e;
  }
  kern<<<(unsigned)(p.groups * p.blocks_per_group), threads, smem, s>>>(p);
  return cudaGetLastError();
}
template <typename T, typename P, int V, int E, int kThreads>
cudaError_t backward_e(const NormBwdParams &p, const NormBwdPlan &plan, cudaStream_t s) {
  return p.post_weight ? backward_post<T, P, V, E, kThreads, true>(p, plan, s)
                       : backward_post<T, P, V, E, kThreads, false>(p, plan, s);
}

template <typename T, typename P>
cudaError_t backward(NormBwdParams p, bool vec, cudaStream_t s, int *launches) {
  const NormBwdPlan plan = norm_bwd_plan(p.rows, p.groups, p.C);
  p.warps_per_row = plan.warps_per_row;
  p.blocks_per_group = plan.blocks_per_group;
  p.rows_per_group = p.rows / p.groups;
  // (blocks of 512 threads leave 128 registers a thread, too few for 16
  // elements: they serve the rows that need them)
  constexpr int V = kVec16<T>;
  cudaError_t e;
  if (vec)
    e = short_rows(p.C)    ? backward_e<T, P, V, 8, 256>(p, plan, s)
        : p.C <= 8 * 512 ? backward_e<T, P, V, 16, 256>(p, plan, s)
                         : backward_e<T, P, V, 16, 512>(p, plan, s);
  else
    e = short_rows(p.C)    ? backward_e<T, P, 1, 8, 256>(p, plan, s)
        : p.C <= 8 * 512 ? backward_e<T, P, 1, 16, 256>(p, plan, s)
                         : backward_e<T, P, 1, 16, 512>(p, plan, s);
  *launches = 1;
  if (e != cudaSuccess || !p.part) return e;
  const unsigned blocks = (unsigned)((p.C + 7) / 8);
  if (p.groups == 1) {
    norm_bwd_sum_kernel<P><<<blocks, p.blocks_per_group > 64 ? 1024 : 256, 0, s>>>(p);
  } else {
    // (up to 64 groups: blocks of 512 threads, several to an SM)
    const int threads = p.groups <= 64 ? 512 : 1024;
    p.share = 1;
    while (2 * p.share * p.groups <= threads / 8) p.share *= 2;
    norm_bwd_groups_kernel<P><<<blocks, threads, 0, s>>>(p);
  }
  ++*launches;
  return cudaGetLastError();
}

}  // namespace

// About 8 warps a block (16 for long rows), and as many blocks as the 148 SMs
// hold at once: two of 256 threads and 128 registers, or one (a block more would
// start when the others end: at 16400 x 1408 in 16 gate groups that took 1.6 times
// as long).  At least one block per gate group.
NormBwdPlan norm_bwd_plan(int64_t rows, int64_t groups, int64_t C) {
  NormBwdPlan plan;
  const bool small = short_rows(C);
  plan.warps_per_row = (int)(small ? (C + 255) / 256 : (C + 511) / 512);
  plan.slots = plan.warps_per_row >= 8 ? 1 : 8 / plan.warps_per_row;
  const int64_t resident = 148 * (small ? 512 / (32 * plan.warps_per_row * plan.slots) : 1);
  const int64_t per_group = (rows / groups + plan.slots - 1) / plan.slots;
  const int64_t share = resident / groups > 1 ? resident / groups : 1;
  plan.blocks_per_group = share < per_group ? share : per_group;
  plan.part_floats = groups * plan.blocks_per_group * 4 * C;
  return plan;
}

int64_t norm_bwd_floats(int64_t rows, int64_t groups, int64_t C) {
  return norm_bwd_plan(rows, groups, C).part_floats;
}

cudaError_t launch_residual_norm(const NormParams &p, int dtype, int param_dtype, bool vec,
                                 cudaStream_t s) {
  if (dtype == SCMP_F32) return forward<float, float>(p, vec, s);
  if (dtype == SCMP_BF16)
    return param_dtype == SCMP_F32 ? forward<__nv_bfloat16, float>(p, vec, s)
                                   : forward<__nv_bfloat16, __nv_bfloat16>(p, vec, s);
  return param_dtype == SCMP_F32 ? forward<__half, float>(p, vec, s)
                                 : forward<__half, __half>(p, vec, s);
}

cudaError_t launch_residual_norm_bwd(const NormBwdParams &p, int dtype, int param_dtype, bool vec,
                                     cudaStream_t s, int *launches) {
  if (dtype == SCMP_F32) return backward<float, float>(p, vec, s, launches);
  if (dtype == SCMP_BF16)
    return param_dtype == SCMP_F32 ? backward<__nv_bfloat16, float>(p, vec, s, launches)
                                   : backward<__nv_bfloat16, __nv_bfloat16>(p, vec, s, launches);
  return param_dtype == SCMP_F32 ? backward<__half, float>(p, vec, s, launches)
                                 : backward<__half, __half>(p, vec, s, launches);
}

}  // namespace scmp
