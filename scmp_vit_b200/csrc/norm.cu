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

// Columns of lane `lane` of warp `w` (of the `G` that share a row), chunk j.
template <int V> __device__ __forceinline__ int col_of(int j, int G, int w, int lane) {
  return ((j * G + w) * 32 + lane) * V;
}

// V consecutive elements at p (16-byte pieces when V > 1).
template <typename T, int V> __device__ __forceinline__ void load_v(const T *p, float *v) {
  if (V == 1) {
    v[0] = to_f32(*p);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += kVec16<T>)
      unpack16<T>(__ldg(reinterpret_cast<const uint4 *>(p + i)), v + i);
  }
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

// Sums over the warps of a row.  Two buffers in turn: a warp writes one again
// only after the barrier that follows every read of it.
struct RowSum {
  float2 *buf;  // [2][warps of the block]
  int warps, first, G, turn;
  __device__ __forceinline__ float2 operator()(float2 v) {
    v = warp_sum(v);
    if (G == 1) return v;
    float2 *b = buf + turn * warps;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
    __syncthreads();
    v = make_float2(0.f, 0.f);
    for (int i = 0; i < G; ++i) {
      v.x += b[first + i].x;
      v.y += b[first + i].y;
    }
    return v;
  }
  __device__ __forceinline__ float operator()(float v) {
    return (*this)(make_float2(v, 0.f)).x;
  }
};

constexpr int kMaxWarps = 16;

// v (valid where in(j)) -> N(v) and its statistics.
template <int NV, int V, typename In>
__device__ __forceinline__ float2 normalise(float (&v)[NV][V], const In &in, RowSum &sum,
                                            float inv_c, float eps, bool rms) {
  float mean = 0.f;
  if (!rms) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[j][i];  // 0 past the row
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
  float amax = 0.f, v8[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v8[i] = i < V ? v[i] : 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) amax = max_nan(amax, fabsf(v[i]));
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) amax = max_nan(amax, __shfl_xor_sync(~0u, amax, o));
  uint32_t codes;
  const uint32_t scale = mx_encode8<kFmt>(v8, amax, 1.0f, &codes);
  if (row < p.rows && col < p.kp) {
    uint8_t *d = p.mx_data + row * (p.kp >> 1) + (col >> 1);
    if (V == 8)
      *reinterpret_cast<uint32_t *>(d) = codes;
    else
      *reinterpret_cast<uint16_t *>(d) = (uint16_t)codes;
  }
  uint32_t word = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    word |= __shfl_sync(~0u, scale, (lane & ~(4 * kLanes - 1)) + b * kLanes) << (8 * b);
  const int64_t g = col / (4 * kBlock);
  if ((lane & (4 * kLanes - 1)) == 0 && g < p.groups)
    *reinterpret_cast<uint32_t *>(p.mx_scales + mx_scale_word(row, g, p.groups)) = word;
}

// G warps per row, 32 elements per lane.
template <typename T, typename P, int V>
__global__ void __launch_bounds__(32 * kMaxWarps)
    residual_norm_kernel(const __grid_constant__ NormParams p) {
  constexpr int NV = 32 / V;
  __shared__ float2 buf[2 * kMaxWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.warps_per_row, w = warp % G;
  RowSum sum{buf, (int)(blockDim.x >> 5), warp - w, G, 0};
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / (32 * G)) + warp / G;
  const bool live = row < p.rows;
  const int C = p.C;
  const float inv_c = 1.0f / (float)C;
  const auto in = [&](int j) { return col_of<V>(j, G, w, lane) < C; };
  const int64_t at = row * C;

  float r[NV][V], z[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = col_of<V>(j, G, w, lane);
#pragma unroll
    for (int i = 0; i < V; ++i) r[j][i] = z[j][i] = 0.f;
    if (live && c < C) {
      load_v<T, V>(static_cast<const T *>(p.x) + at + c, r[j]);
      if (p.y) load_v<T, V>(static_cast<const T *>(p.y) + at + c, z[j]);
    }
  }
  if (p.y) {
    if (p.post_weight) {
      const float2 st = normalise<NV, V>(z, in, sum, inv_c, p.eps, p.rms);
      if (p.stats && live && w == 0 && lane == 0) p.stats[p.rows + row] = st;
    }
    const int64_t gate_at = p.gate && live ? row / p.rows_per_gate * C : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col_of<V>(j, G, w, lane);
      if (!live || c >= C) continue;
      float f[V], g[V];
      if (p.post_weight) {
        load_v<P, V>(static_cast<const P *>(p.post_weight) + c, f);
#pragma unroll
        for (int i = 0; i < V; ++i) z[j][i] *= f[i];
        if (p.post_bias) {
          load_v<P, V>(static_cast<const P *>(p.post_bias) + c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) z[j][i] += f[i];
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
      // r is rounded to its type once, and the norm sees the rounded value: the
      // one that the next block and the backward pass read
#pragma unroll
      for (int i = 0; i < V; ++i)
        r[j][i] = to_f32(from_f32<T>(__fmaf_rn(z[j][i], f[i], r[j][i])));
      store_v<T, V>(static_cast<T *>(p.r) + at + c, r[j]);
    }
  }
  const float2 st = normalise<NV, V>(r, in, sum, inv_c, p.eps, p.rms);
  if (p.stats && live && w == 0 && lane == 0) p.stats[row] = st;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = col_of<V>(j, G, w, lane);
    if (live && c < C) {
      float f[V];
      load_v<P, V>(static_cast<const P *>(p.weight) + c, f);
#pragma unroll
      for (int i = 0; i < V; ++i) r[j][i] *= f[i];
      if (p.bias) {
        load_v<P, V>(static_cast<const P *>(p.bias) + c, f);
#pragma unroll
        for (int i = 0; i < V; ++i) r[j][i] += f[i];
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

// ---------------------------------------------------------------- backward
// Rows of one gate group (all rows without a gate) are dealt to `per_group`
// row slots; a slot is G warps with 16 elements per lane, a block holds a few
// slots of one group.  Column sums stay in registers over a slot's rows, are
// added over the block's slots in shared memory in a fixed order and written
// as partials [group][block][part][C]; a second kernel adds those in order, so
// the result does not depend on timing.
//   parts: 0 sum dh n   1 sum dh   2 sum g z (no post norm) or sum g m   3 sum g
template <typename T, typename P, int V, bool kPost>
__global__ void __launch_bounds__(32 * kMaxWarps)
    residual_norm_bwd_kernel(const __grid_constant__ NormBwdParams p) {
  constexpr int NV = 16 / V;
  constexpr int kParts = kPost ? 4 : 3;
  __shared__ float2 buf[2 * kMaxWarps];
  extern __shared__ float part_smem[];  // [C], blocks of several slots
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.warps_per_row, w = warp % G, slot = warp / G;
  const int slots = blockDim.x / (32 * G);
  RowSum sum{buf, (int)(blockDim.x >> 5), warp - w, G, 0};
  const int C = p.C;
  const float inv_c = 1.0f / (float)C;
  const int64_t group = blockIdx.x / p.blocks_per_group;
  const int64_t first = (blockIdx.x % p.blocks_per_group) * slots + slot;
  const int64_t stride = p.blocks_per_group * slots;

  float acc[kParts][NV][V];
#pragma unroll
  for (int k = 0; k < kParts; ++k)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[k][j][i] = 0.f;

  // every slot of a block runs the same number of rounds: the row sums meet at
  // block barriers
  const int64_t rounds = (p.rows_per_group + stride - 1) / stride;
  for (int64_t t = 0; t < rounds; ++t) {
    const int64_t in_group = first + t * stride;
    const bool live = in_group < p.rows_per_group;
    const int64_t row = group * p.rows_per_group + in_group;
    const int64_t at = row * C;
    float n[NV][V], g[NV][V], dn[NV][V], y[NV][V];
    float2 st = make_float2(0.f, 0.f), st_y = st;
    if (live) {
      st = p.stats[row];
      if (kPost) st_y = p.stats[p.rows + row];
    }
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col_of<V>(j, G, w, lane);
#pragma unroll
      for (int i = 0; i < V; ++i) n[j][i] = g[j][i] = dn[j][i] = y[j][i] = 0.f;
      if (!live || c >= C) continue;
      load_v<T, V>(static_cast<const T *>(p.r) + at + c, n[j]);
      if (p.dh) load_v<T, V>(static_cast<const T *>(p.dh) + at + c, dn[j]);
      if (p.dr) load_v<T, V>(static_cast<const T *>(p.dr) + at + c, g[j]);
      if (p.y) load_v<T, V>(static_cast<const T *>(p.y) + at + c, y[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col_of<V>(j, G, w, lane);
      if (!live || c >= C) continue;
      float f[V];
      load_v<P, V>(static_cast<const P *>(p.weight) + c, f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        n[j][i] = (n[j][i] - st.x) * st.y;
        acc[0][j][i] = __fmaf_rn(dn[j][i], n[j][i], acc[0][j][i]);
        acc[1][j][i] += dn[j][i];
        dn[j][i] *= f[i];
        s.x += dn[j][i];
        s.y = __fmaf_rn(dn[j][i], n[j][i], s.y);
      }
    }
    s = sum(s);
    const float mean_dn = p.rms ? 0.f : s.x * inv_c, mean_dnn = s.y * inv_c;
    float2 s2 = make_float2(0.f, 0.f);
    const int64_t gate_at = group * C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col_of<V>(j, G, w, lane);
      if (!live || c >= C) continue;
#pragma unroll
      for (int i = 0; i < V; ++i)
        g[j][i] = __fmaf_rn(st.y, __fmaf_rn(-n[j][i], mean_dnn, dn[j][i] - mean_dn), g[j][i]);
      if (p.dx) store_v<T, V>(static_cast<T *>(p.dx) + at + c, g[j]);
      if (!p.y) continue;
      float f[V], e[V];
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = 1.0f;
      if (p.gamma) load_v<P, V>(static_cast<const P *>(p.gamma) + c, f);
      if (p.gate) {
        load_v<P, V>(static_cast<const P *>(p.gate) + gate_at + c, e);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] *= e[i];
      }
      if (kPost) {
        load_v<P, V>(static_cast<const P *>(p.post_weight) + c, e);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          y[j][i] = (y[j][i] - st_y.x) * st_y.y;
          acc[2][j][i] = __fmaf_rn(g[j][i], y[j][i], acc[2][j][i]);
          acc[kParts - 1][j][i] += g[j][i];
          dn[j][i] = g[j][i] * f[i] * e[i];
          s2.x += dn[j][i];
          s2.y = __fmaf_rn(dn[j][i], y[j][i], s2.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          acc[2][j][i] = __fmaf_rn(g[j][i], y[j][i], acc[2][j][i]);
          dn[j][i] = g[j][i] * f[i];
        }
        if (p.dy) store_v<T, V>(static_cast<T *>(p.dy) + at + c, dn[j]);
      }
    }
    if (kPost) {
      s2 = sum(s2);
      const float mean_dm = p.rms ? 0.f : s2.x * inv_c, mean_dmm = s2.y * inv_c;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = col_of<V>(j, G, w, lane);
        if (!live || c >= C || !p.dy) continue;
#pragma unroll
        for (int i = 0; i < V; ++i)
          dn[j][i] = st_y.y * __fmaf_rn(-y[j][i], mean_dmm, dn[j][i] - mean_dm);
        store_v<T, V>(static_cast<T *>(p.dy) + at + c, dn[j]);
      }
    }
  }
  if (!p.part) return;
  float *out = p.part + (int64_t)blockIdx.x * 4 * C;
#pragma unroll
  for (int k = 0; k < kParts; ++k) {
    for (int q = slots - 1; q > 0; --q) {  // slot q adds to what q + 1.. left; slot 0 writes
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

// Block (32 columns, gate group): 32 warps share the group's partials.  With
// one group it finishes; else it leaves the group's sums for the kernel below.
template <typename P>
__global__ void __launch_bounds__(1024) norm_bwd_sum_kernel(
    const __grid_constant__ NormBwdParams p) {
  __shared__ float s[4][32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cols = (p.C + 31) / 32;
  const int c = (int)(blockIdx.x % cols) * 32 + lane;
  const int64_t group = blockIdx.x / cols;
  const int parts = p.post_weight ? 4 : 3;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < p.C)
    for (int64_t b = warp; b < p.blocks_per_group; b += 32) {
      const float *src = p.part + (group * p.blocks_per_group + b) * 4 * p.C + c;
      for (int k = 0; k < parts; ++k) v[k] += src[(int64_t)k * p.C];
    }
#pragma unroll
  for (int k = 0; k < 4; ++k) s[k][warp][lane] = v[k];
  __syncthreads();
  if (warp < 4) {
    float t = 0.f;
    for (int i = 0; i < 32; ++i) t += s[warp][i][lane];
    if (p.groups > 1 && c < p.C) p.sums[(group * 4 + warp) * p.C + c] = t;
    s[warp][0][lane] = t;  // read above by this thread alone
  }
  if (p.groups > 1) return;
  __syncthreads();
  if (warp == 0 && c < p.C) {
    const float one[4] = {s[0][0][lane], s[1][0][lane], s[2][0][lane], s[3][0][lane]};
    float total[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
    add_group<P>(p, 0, c, one, total);
    write_totals<P>(p, c, total);
  }
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

template <typename T, typename P>
cudaError_t forward(NormParams p, bool vec, cudaStream_t s) {
  constexpr int V = kVec16<T>;
  const int G = (p.C + 1023) / 1024;  // 32 elements per lane
  const int rows_per_block = G >= 4 ? 1 : 4 / G;
  p.warps_per_row = G;
  const int64_t rows = p.mx_data ? (p.rows + 127) / 128 * 128 : p.rows;
  const int64_t blocks = (rows + rows_per_block - 1) / rows_per_block;
  const int threads = 32 * G * rows_per_block;
  if (vec)
    residual_norm_kernel<T, P, V><<<(unsigned)blocks, threads, 0, s>>>(p);
  else
    residual_norm_kernel<T, P, 1><<<(unsigned)blocks, threads, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, typename P, int V>
cudaError_t backward_v(const NormBwdParams &p, const NormBwdPlan &plan, cudaStream_t s) {
  const size_t smem = plan.slots > 1 ? (size_t)p.C * sizeof(float) : 0;
  const unsigned blocks = (unsigned)(p.groups * p.blocks_per_group);
  const int threads = 32 * plan.warps_per_row * plan.slots;
  if (p.post_weight)
    residual_norm_bwd_kernel<T, P, V, true><<<blocks, threads, smem, s>>>(p);
  else
    residual_norm_bwd_kernel<T, P, V, false><<<blocks, threads, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, typename P>
cudaError_t backward(NormBwdParams p, bool vec, cudaStream_t s, int *launches) {
  const NormBwdPlan plan = norm_bwd_plan(p.rows, p.groups, p.C);
  p.warps_per_row = plan.warps_per_row;
  p.blocks_per_group = plan.blocks_per_group;
  p.rows_per_group = p.rows / p.groups;
  if (!p.part_needed) p.part = nullptr;
  cudaError_t e = vec ? backward_v<T, P, kVec16<T>>(p, plan, s) : backward_v<T, P, 1>(p, plan, s);
  *launches = 1;
  if (e != cudaSuccess || !p.part) return e;
  const unsigned cols = (unsigned)((p.C + 31) / 32);
  norm_bwd_sum_kernel<P><<<(unsigned)(cols * p.groups), 1024, 0, s>>>(p);
  ++*launches;
  if ((e = cudaGetLastError()) != cudaSuccess || p.groups == 1) return e;
  norm_bwd_groups_kernel<P><<<cols, 1024, 0, s>>>(p);
  ++*launches;
  return cudaGetLastError();
}

}  // namespace

// Slots of 16 elements per lane, about 8 warps a block, and two blocks on each
// of the 148 SMs in all (at least one block per gate group).
NormBwdPlan norm_bwd_plan(int64_t rows, int64_t groups, int64_t C) {
  NormBwdPlan plan;
  plan.warps_per_row = (int)((C + 511) / 512);
  plan.slots = plan.warps_per_row >= 8 ? 1 : 8 / plan.warps_per_row;
  const int64_t per_group = (rows / groups + plan.slots - 1) / plan.slots;
  const int64_t want = (2 * 148 + groups - 1) / groups;
  plan.blocks_per_group = want < per_group ? want : per_group;
  plan.part_floats = groups * plan.blocks_per_group * 4 * C;
  plan.sum_floats = groups > 1 ? groups * 4 * C : 0;
  return plan;
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
