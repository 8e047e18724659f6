// Gated residual add with the norms around it, in one pass over the rows, and
// its gradients:
//   z = y, or N(y) pw + pb (a norm behind the branch)
//   r = x + z gamma gate          rounded to x's type
//   h = N(r) w + b                the norm in front of the next branch
// N(v) = (v - mean) / sqrt(var + eps), or v / sqrt(mean v^2 + eps).  A row stays
// in registers from its loads to its stores; statistics are fp32, the variance
// a second pass over the registers.
#include "norm.cuh"

#include "mx_common.cuh"

namespace scmp {
namespace {

// A row is dealt to G warps: chunk j (of V consecutive columns per lane) of warp
// w starts at column ((j G + w) 32 + lane) V.
template <int V> __device__ __forceinline__ int col_of(int j, int G, int w, int lane) {
  return ((j * G + w) * 32 + lane) * V;
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

__device__ __forceinline__ float2 warp_sum(float2 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(~0u, v.x, o);
    v.y += __shfl_xor_sync(~0u, v.y, o);
  }
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

constexpr int kMaxWarps = 16;

// Sums over the G warps of a row slot, which meet at a barrier of their own.
// Two buffers in turn: a warp writes one again only after the barrier that
// follows every read of it.
struct RowSum {
  float2 *buf;  // this slot's warps in [2][kMaxWarps]
  int G, w, barrier, turn;
  __device__ RowSum(float2 *all, int G_, int slot, int w_)
      : buf(all + slot * G_), G(G_), w(w_), barrier(1 + slot), turn(0) {}
  __device__ __forceinline__ float2 meet(float2 v) {
    float2 *b = buf + turn * kMaxWarps;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) b[w] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(G * 32) : "memory");
    v = make_float2(0.f, 0.f);
    for (int i = 0; i < G; ++i) {
      v.x += b[i].x;
      v.y += b[i].y;
    }
    return v;
  }
  __device__ __forceinline__ float2 operator()(float2 v) {
    v = warp_sum(v);
    return G == 1 ? v : meet(v);
  }
  __device__ __forceinline__ float operator()(float v) {
    v = warp_sum(v);
    return G == 1 ? v : meet(make_float2(v, 0.f)).x;
  }
};

// v (0 past the row, where in(j) is false) -> N(v) and its statistics.
template <int NV, int V, typename In>
__device__ __forceinline__ float2 normalise(float (&v)[NV][V], const In &in, RowSum &sum,
                                            float inv_c, float eps, bool rms) {
  float mean = 0.f;
  if (!rms) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[j][i];
    mean = sum(s) * inv_c;
  }
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[j][i] = in(j) ? v[j][i] - mean : 0.f;
      q = __fmaf_rn(v[j][i], v[j][i], q);
    }
  const float rstd = 1.0f / sqrtf(__fmaf_rn(sum(q), inv_c, eps));
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) v[j][i] *= rstd;
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
//           warps an SM.  Few rows (257 x 1024: 3.3, E = 16 3.5), fp32 (16448 x
//           1024: 49.7 = a copy's rate, E = 16 57.9), short rows (16448 x 200:
//           9.1, E = 16 10.7)
//   E = 16  slots walk rows, and once a row's x and y are used the next one is on
//           its way into their registers.  Many rows (16448 x 1024: 30.6, E = 8
//           42.1)
//   E = 32  the same for rows of over 4096 columns, or not in 16-byte pieces
template <typename T, typename P, int V, int E>
__global__ void __launch_bounds__(256, E == 16 ? 3 : 1)
    residual_norm_kernel(const __grid_constant__ NormParams p) {
  constexpr bool kWalk = E > 8;
  constexpr int NV = E / V;
  __shared__ float2 buf[2 * kMaxWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.warps_per_row, slot = warp / G, w = warp - slot * G;
  const int slots = blockDim.x / (32 * G);
  RowSum sum(buf, G, slot, w);
  const int C = p.C;
  const float inv_c = 1.0f / (float)C;
  const auto in_row = [&](int j) { return col_of<V>(j, G, w, lane) < C; };

  Pack<T, V> x[NV], y[NV];
  const auto load = [&](int64_t row) {
    const bool live = row < p.rows;
    const int64_t at = row * C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x[j].zero();
      y[j].zero();
      if (!live || !in_row(j)) continue;
      const int c = col_of<V>(j, G, w, lane);
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
    float r[NV][V];
    if (p.y) {
#pragma unroll
      for (int j = 0; j < NV; ++j) y[j].get(r[j]);
      if (p.post_weight) {
        const float2 st = normalise<NV, V>(r, in, sum, inv_c, p.eps, p.rms);
        if (p.stats && live && w == 0 && lane == 0) p.stats[p.rows + row] = st;
      }
      const int64_t gate_at = p.gate && live ? row / p.rows_per_gate * C : 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = col_of<V>(j, G, w, lane);
        if (!in(j)) {
#pragma unroll
          for (int i = 0; i < V; ++i) r[j][i] = 0.f;
          continue;
        }
        float f[V], g[V];
        if (p.post_weight) {
          load_v<P, V>(static_cast<const P *>(p.post_weight) + c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) r[j][i] *= f[i];
          if (p.post_bias) {
            load_v<P, V>(static_cast<const P *>(p.post_bias) + c, f);
#pragma unroll
            for (int i = 0; i < V; ++i) r[j][i] += f[i];
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = 1.0f;
        if (p.gamma) load_v<P, V>(static_cast<const P *>(p.gamma) + c, f);
        if (p.gate) {
          load_v<P, V>(static_cast<const P *>(p.gate) + gate_at + c, g);
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] *= g[i];
        }
        x[j].get(g);
        // r is rounded to its type once, and the norm sees the rounded value:
        // the one that the next block and the backward pass read
#pragma unroll
        for (int i = 0; i < V; ++i)
          r[j][i] = to_f32(from_f32<T>(__fmaf_rn(r[j][i], f[i], g[i])));
        store_v<T, V>(static_cast<T *>(p.r) + at + c, r[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) x[j].get(r[j]);
    }
    if (kWalk) load(row + stride);
    const float2 st = normalise<NV, V>(r, in, sum, inv_c, p.eps, p.rms);
    if (p.stats && live && w == 0 && lane == 0) p.stats[row] = st;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col_of<V>(j, G, w, lane);
      if (in(j)) {
        float f[V], g[V];
        load_v<P, V>(static_cast<const P *>(p.weight) + c, f);
        if (p.bias) {
          load_v<P, V>(static_cast<const P *>(p.bias) + c, g);
#pragma unroll
          for (int i = 0; i < V; ++i) r[j][i] = __fmaf_rn(r[j][i], f[i], g[i]);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) r[j][i] *= f[i];
        }
        if (p.h) {
          if (p.h_f32)
            store_v<float, V>(static_cast<float *>(p.h) + at + c, r[j]);
          else
            store_v<T, V>(static_cast<T *>(p.h) + at + c, r[j]);
        }
      }
      if (V > 1 && p.mx_data) {
        if (p.fmt == SCMP_MXFP4)
          store_mx<SCMP_MXFP4, V>(p, r[j], row, c, lane);
        else
          store_mx<SCMP_NVFP4, V>(p, r[j], row, c, lane);
      }
    }
  }
}

// ---------------------------------------------------------------- backward
// Rows of one gate group (all rows without a gate) are dealt to row slots of G
// warps; a block holds a few slots of one group.  While a row is worked on, the
// slot's next row is on its way into registers.  Column sums stay in registers
// over a slot's rows, are added over the block's slots in shared memory in a
// fixed order and written as partials [group][block][part][C]; a second kernel
// adds those in order, so the result does not depend on timing.
//   parts: 0 sum dh n   1 sum dh   2 sum g z (no post norm) or sum g m   3 sum g
// E = 8 elements per lane for rows of up to 2048 in 16-byte pieces, else 16.
template <typename T, int V, int NV> struct BwdRow {
  Pack<T, V> r[NV], y[NV], dr[NV], dh[NV];
  float2 st, st_y;
};
template <typename T, int V, int NV>
__device__ __forceinline__ void load_row(const NormBwdParams &p, int64_t row, bool live, int G,
                                         int w, int lane, bool post, BwdRow<T, V, NV> &q) {
  q.st = q.st_y = make_float2(0.f, 0.f);
  if (live) {
    q.st = p.stats[row];
    if (post) q.st_y = p.stats[p.rows + row];
  }
  const int64_t at = row * p.C;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = col_of<V>(j, G, w, lane);
    q.r[j].zero();
    q.y[j].zero();
    q.dr[j].zero();
    q.dh[j].zero();
    if (!live || c >= p.C) continue;
    q.r[j].load(static_cast<const T *>(p.r) + at + c);
    if (p.dh) q.dh[j].load(static_cast<const T *>(p.dh) + at + c);
    if (p.dr) q.dr[j].load(static_cast<const T *>(p.dr) + at + c);
    if (p.y) q.y[j].load(static_cast<const T *>(p.y) + at + c);
  }
}

template <typename T, typename P, int V, int E, bool kPost, int kThreads>
__global__ void __launch_bounds__(kThreads, E == 8 ? 2 : 1)
    residual_norm_bwd_kernel(const __grid_constant__ NormBwdParams p) {
  constexpr int NV = E / V;
  constexpr int kParts = kPost ? 4 : 3;
  __shared__ float2 buf[2 * kMaxWarps];
  extern __shared__ float part_smem[];  // [C], blocks of several slots
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.warps_per_row, slot = warp / G, w = warp - slot * G;
  const int slots = blockDim.x / (32 * G);
  RowSum sum(buf, G, slot, w);
  const int C = p.C;
  const float inv_c = 1.0f / (float)C;
  const int64_t group = blockIdx.x / p.blocks_per_group;
  const int64_t stride = p.blocks_per_group * slots;
  const int64_t row0 = group * p.rows_per_group;

  // the parameters of this lane's columns stay the same over the rows
  float wt[NV][V], sc[NV][V], pw[kPost ? NV : 1][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = col_of<V>(j, G, w, lane);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      wt[j][i] = 0.f;
      sc[j][i] = 1.f;
      if (kPost) pw[kPost ? j : 0][i] = 0.f;
    }
    if (c >= C) continue;
    load_v<P, V>(static_cast<const P *>(p.weight) + c, wt[j]);
    if (p.gamma) load_v<P, V>(static_cast<const P *>(p.gamma) + c, sc[j]);
    if (p.gate) {
      float g[V];
      load_v<P, V>(static_cast<const P *>(p.gate) + group * C + c, g);
#pragma unroll
      for (int i = 0; i < V; ++i) sc[j][i] *= g[i];
    }
    if (kPost) load_v<P, V>(static_cast<const P *>(p.post_weight) + c, pw[kPost ? j : 0]);
  }
  float acc[kParts][NV][V];
#pragma unroll
  for (int k = 0; k < kParts; ++k)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[k][j][i] = 0.f;

  int64_t i_row = (blockIdx.x % p.blocks_per_group) * slots + slot;
  BwdRow<T, V, NV> next;
  load_row<T, V, NV>(p, row0 + i_row, i_row < p.rows_per_group, G, w, lane, kPost, next);
  for (; i_row < p.rows_per_group; i_row += stride) {
    const BwdRow<T, V, NV> q = next;
    load_row<T, V, NV>(p, row0 + i_row + stride, i_row + stride < p.rows_per_group, G, w, lane,
                       kPost, next);
    const int64_t at = (row0 + i_row) * C;
    float n[NV][V], dn[NV][V];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool in = col_of<V>(j, G, w, lane) < C;
      q.r[j].get(n[j]);
      q.dh[j].get(dn[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        n[j][i] = in ? (n[j][i] - q.st.x) * q.st.y : 0.f;
        acc[0][j][i] = __fmaf_rn(dn[j][i], n[j][i], acc[0][j][i]);
        acc[1][j][i] += dn[j][i];
        dn[j][i] *= wt[j][i];
        s.x += dn[j][i];
        s.y = __fmaf_rn(dn[j][i], n[j][i], s.y);
      }
    }
    s = sum(s);
    const float mean_dn = p.rms ? 0.f : s.x * inv_c, mean_dnn = s.y * inv_c;
    float2 s2 = make_float2(0.f, 0.f);
    float m[kPost ? NV : 1][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col_of<V>(j, G, w, lane);
      float g[V], y[V];
      q.dr[j].get(g);
      q.y[j].get(y);
#pragma unroll
      for (int i = 0; i < V; ++i)
        g[i] = __fmaf_rn(q.st.y, __fmaf_rn(-n[j][i], mean_dnn, dn[j][i] - mean_dn), g[i]);
      if (p.dx && c < C) store_v<T, V>(static_cast<T *>(p.dx) + at + c, g);
      if (kPost) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float mi = c < C ? (y[i] - q.st_y.x) * q.st_y.y : 0.f;
          m[kPost ? j : 0][i] = mi;
          acc[2][j][i] = __fmaf_rn(g[i], mi, acc[2][j][i]);
          acc[kParts - 1][j][i] += g[i];
          dn[j][i] = g[i] * sc[j][i] * pw[kPost ? j : 0][i];
          s2.x += dn[j][i];
          s2.y = __fmaf_rn(dn[j][i], mi, s2.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          acc[2][j][i] = __fmaf_rn(g[i], y[i], acc[2][j][i]);
          g[i] *= sc[j][i];
        }
        if (p.dy && c < C) store_v<T, V>(static_cast<T *>(p.dy) + at + c, g);
      }
    }
    if (kPost) {
      s2 = sum(s2);
      const float mean_dm = p.rms ? 0.f : s2.x * inv_c, mean_dmm = s2.y * inv_c;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = col_of<V>(j, G, w, lane);
        if (c >= C || !p.dy) continue;
#pragma unroll
        for (int i = 0; i < V; ++i)
          dn[j][i] = q.st_y.y * __fmaf_rn(-m[kPost ? j : 0][i], mean_dmm, dn[j][i] - mean_dm);
        store_v<T, V>(static_cast<T *>(p.dy) + at + c, dn[j]);
      }
    }
  }
  if (!p.part) return;
  float *out = p.part + (int64_t)blockIdx.x * 4 * C;
#pragma unroll
  for (int k = 0; k < kParts; ++k) {
    for (int q = slots - 1; q > 0; --q) {  // the slots add up, from the last to the first
      __syncthreads();
      if (slot == q) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int c = col_of<V>(j, G, w, lane);
          if (c >= C) continue;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float v = acc[k][j][i];
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
        const int c = col_of<V>(j, G, w, lane);
        if (c >= C) continue;
#pragma unroll
        for (int i = 0; i < V; ++i)
          out[(int64_t)k * C + c + i] = acc[k][j][i] + (slots > 1 ? part_smem[c + i] : 0.f);
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

// Block (8 columns, gate group): 32 or 128 threads per column share the group's
// partials.  With one group it finishes; else it leaves the group's sums for the
// kernel below.
template <typename P>
__global__ void __launch_bounds__(1024) norm_bwd_sum_kernel(
    const __grid_constant__ NormBwdParams p) {
  __shared__ float s[4][32][8];
  const int cols = (p.C + 7) / 8;
  const int ci = threadIdx.x & 7, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (int)(blockIdx.x % cols) * 8 + ci;
  const int64_t group = blockIdx.x / cols;
  const int parts = p.post_weight ? 4 : 3;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < p.C)
    for (int64_t b = threadIdx.x >> 3; b < p.blocks_per_group; b += blockDim.x >> 3) {
      const float *src = p.part + (group * p.blocks_per_group + b) * 4 * p.C + c;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < parts) v[k] += src[(int64_t)k * p.C];
    }
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
    if (p.groups > 1) p.sums[(group * 4 + k) * p.C + c] = one[k];
  }
  if (p.groups > 1) return;
  float total[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  add_group<P>(p, 0, c, one, total);
  write_totals<P>(p, c, total);
}

template <typename P>
__global__ void __launch_bounds__(1024) norm_bwd_groups_kernel(
    const __grid_constant__ NormBwdParams p) {
  __shared__ float s[5][32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float total[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  if (c < p.C)
    for (int64_t g = warp; g < p.groups; g += 32) {
      float one[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) one[k] = p.sums[(g * 4 + k) * p.C + c];
      add_group<P>(p, g, c, one, total);
    }
#pragma unroll
  for (int k = 0; k < 5; ++k) s[k][warp][lane] = total[k];
  __syncthreads();
  if (warp == 0 && c < p.C) {
#pragma unroll
    for (int k = 0; k < 5; ++k) {
      total[k] = 0.f;
      for (int i = 0; i < 32; ++i) total[k] += s[k][i][lane];
    }
    write_totals<P>(p, c, total);
  }
}

// --------------------------------------------------------------- dispatch

// Backward: elements per lane, 8 for rows of up to 2048 in 16-byte pieces.
bool short_rows(int64_t C, bool vec) { return vec && C <= 2048; }

template <typename T, typename P, int V, int E>
cudaError_t forward_e(NormParams p, cudaStream_t s) {
  const int G = (p.C + 32 * E - 1) / (32 * E), slots = 8 / G, threads = 32 * G * slots;
  p.warps_per_row = G;
  p.row_end = p.mx_data ? (p.rows + 127) / 128 * 128 : p.rows;
  const int64_t blocks = (p.row_end + slots - 1) / slots;
  // walking slots: the blocks that 148 SMs hold at once
  const int64_t most = E == 8 ? blocks : 148 * ((E == 16 ? 768 : 512) / threads);
  residual_norm_kernel<T, P, V, E>
      <<<(unsigned)(blocks < most ? blocks : most), threads, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, typename P>
cudaError_t forward(const NormParams &p, bool vec, cudaStream_t s) {
  constexpr int V = kVec16<T>;
  if (!vec) return forward_e<T, P, 1, 32>(p, s);
  if (p.C <= 256 || (p.C <= 2048 && (sizeof(T) == 4 || p.rows <= 148 * 8)))
    return forward_e<T, P, V, 8>(p, s);
  return p.C <= 4096 ? forward_e<T, P, V, 16>(p, s) : forward_e<T, P, V, 32>(p, s);
}

template <typename T, typename P, int V, int E, int kThreads>
cudaError_t backward_e(const NormBwdParams &p, const NormBwdPlan &plan, cudaStream_t s) {
  const size_t smem = plan.slots > 1 ? (size_t)p.C * sizeof(float) : 0;
  const unsigned blocks = (unsigned)(p.groups * p.blocks_per_group);
  const int threads = 32 * plan.warps_per_row * plan.slots;
  if (p.post_weight)
    residual_norm_bwd_kernel<T, P, V, E, true, kThreads><<<blocks, threads, smem, s>>>(p);
  else
    residual_norm_bwd_kernel<T, P, V, E, false, kThreads><<<blocks, threads, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, typename P>
cudaError_t backward(NormBwdParams p, bool vec, cudaStream_t s, int *launches) {
  const NormBwdPlan plan = norm_bwd_plan(p.rows, p.groups, p.C, vec);
  p.warps_per_row = plan.warps_per_row;
  p.blocks_per_group = plan.blocks_per_group;
  p.rows_per_group = p.rows / p.groups;
  p.sums = p.part ? p.part + plan.part_floats : nullptr;
  // (blocks of 512 threads leave 128 registers a thread, too few for 16
  // elements: they serve the rows that need them)
  constexpr int V = kVec16<T>;
  cudaError_t e = short_rows(p.C, vec)    ? backward_e<T, P, V, 8, 256>(p, plan, s)
                  : vec && p.C <= 8 * 512 ? backward_e<T, P, V, 16, 256>(p, plan, s)
                  : vec                   ? backward_e<T, P, V, 16, 512>(p, plan, s)
                                          : backward_e<T, P, 1, 16, 512>(p, plan, s);
  *launches = 1;
  if (e != cudaSuccess || !p.part) return e;
  if (p.groups > 1 && p.blocks_per_group == 1) {
    p.sums = p.part;  // one block per group: its partials are the group's sums
    norm_bwd_groups_kernel<P><<<(unsigned)((p.C + 31) / 32), 1024, 0, s>>>(p);
    ++*launches;
    return cudaGetLastError();
  }
  norm_bwd_sum_kernel<P><<<(unsigned)((p.C + 7) / 8 * p.groups),
                           p.blocks_per_group > 64 ? 1024 : 256, 0, s>>>(p);
  ++*launches;
  if ((e = cudaGetLastError()) != cudaSuccess || p.groups == 1) return e;
  norm_bwd_groups_kernel<P><<<(unsigned)((p.C + 31) / 32), 1024, 0, s>>>(p);
  ++*launches;
  return cudaGetLastError();
}

}  // namespace

// About 8 warps a block (16 for long rows), and as many blocks as the 148 SMs
// hold at once: two of 256 threads and 128 registers, or one (a block more would
// start when the others end: 16400 x 1408 in 16 gate groups 168 us instead of
// 103).  At least one block per gate group.
NormBwdPlan norm_bwd_plan(int64_t rows, int64_t groups, int64_t C, bool vec) {
  NormBwdPlan plan;
  const bool small = short_rows(C, vec);
  plan.warps_per_row = (int)(small ? (C + 255) / 256 : (C + 511) / 512);
  plan.slots = plan.warps_per_row >= 8 ? 1 : 8 / plan.warps_per_row;
  const int64_t resident = 148 * (small ? 512 / (32 * plan.warps_per_row * plan.slots) : 1);
  const int64_t per_group = (rows / groups + plan.slots - 1) / plan.slots;
  const int64_t share = resident / groups > 1 ? resident / groups : 1;
  plan.blocks_per_group = share < per_group ? share : per_group;
  plan.part_floats = groups * plan.blocks_per_group * 4 * C;
  plan.sum_floats = groups > 1 && plan.blocks_per_group > 1 ? groups * 4 * C : 0;
  return plan;
}

int64_t norm_bwd_floats(int64_t rows, int64_t groups, int64_t C) {
  const NormBwdPlan a = norm_bwd_plan(rows, groups, C, true);
  const NormBwdPlan b = norm_bwd_plan(rows, groups, C, false);
  return (a.part_floats > b.part_floats ? a.part_floats : b.part_floats) +
         (a.sum_floats > b.sum_floats ? a.sum_floats : b.sum_floats);
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
