// The fused qkv projection output split into q, k and v with every head's row of q
// and k normalised and turned by multi-axis rotary positions, and its gradients.
//   n = (u - mean) / sqrt(var + eps)  or  u / sqrt(mean u^2 + eps)     over D
//   q = R(n w + b)                    R: the rotation of rotary.cu, rounded once
//   dt = R^T dq,  dw = sum dt n,  db = sum dt,  g = dt w
//   du = (g - mean(g) - n mean(g n)) / sqrt(var + eps)     (rms: without mean(g))
// Statistics are fp32 and not stored: the backward pass reads u in any case.
//
// A group of 1 to 32 lanes owns a token and walks its heads: cos, sin and the
// weights stay in registers, a head's row is one piece per lane, sums over the
// row are shuffles inside the group, and a few heads are in flight at a time.  The
// partner of a pair half a section apart is loaded again (from L1) and normalised
// by its own weight.  HBM-bound: each element is read once and written once.
#include "mx_common.cuh"
#include "qknorm.cuh"
#include "rotary_device.cuh"

namespace scmp {
namespace {

constexpr int kMaxD = 256;

// What a thread holds of one head row: kP pieces of V elements, piece i at element
// (lane + i lanes) V of D.
template <int V, int kP> struct Mine {
  int e0[kP], partner[kP];
  uint32_t mask[kP];  // elements that turn
  bool in[kP];
  float c[kP][V], s[kP][V];
};

template <int V, int kP, bool kInterleaved, bool kBackward>
__device__ __forceinline__ void set_up(const QkNormParams &p, uint32_t tok, uint32_t n, bool turns,
                                       Mine<V, kP> &m) {
  const int lane = threadIdx.x & (p.lanes - 1);
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    m.e0[i] = (lane + i * p.lanes) * V;
    m.in[i] = m.e0[i] < p.r.D;
    m.mask[i] = 0;
    m.partner[i] = m.e0[i];
    if (turns && m.in[i])
      m.mask[i] = angles_of<V, kInterleaved, kBackward>(p.r, p.r.pos_batched ? tok : n, m.e0[i],
                                                        m.c[i], m.s[i], m.partner[i]);
  }
}

// Sums over a group of lanes, of several values at a time.
template <int A> __device__ __forceinline__ void group_sum(int lanes, float (&v)[A]) {
  for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int q = 0; q < A; ++q) v[q] += __shfl_xor_sync(~0u, v[q], o);
}

template <typename T, int V> __device__ __forceinline__ void zero(Piece<T, V> &x) {
  if constexpr (V == 1) {
    x.u[0] = from_f32<T>(0.0f);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T, V>::kWords; ++i) x.u[i] = 0;
  }
}
template <typename T, int V> __device__ __forceinline__ void values(const Piece<T, V> &x, float *v) {
  if constexpr (V == 1)
    v[0] = to_f32(x.u[0]);
  else
    x.get(v);
}
template <typename T, int V> __device__ __forceinline__ void store(T *p, const float *v) {
  Piece<T, V> x;
  if constexpr (V == 1) {
    x.u[0] = from_f32<T>(v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T, V>::kWords; ++i) x.u[i] = Piece<T, V>::word(v, i);
  }
  x.store(p);
}

// mean and 1 / deviation of A head rows (mean 0 for rms).
template <typename T, int V, int kP, int A>
__device__ __forceinline__ void statistics(const QkNormParams &p, const Piece<T, V> (&x)[A][kP],
                                           const Mine<V, kP> &m, float (&mean)[A],
                                           float (&rstd)[A]) {
  const float inv = 1.0f / (float)p.r.D;
#pragma unroll
  for (int q = 0; q < A; ++q) mean[q] = 0.0f;
  if (!p.rms) {
#pragma unroll
    for (int q = 0; q < A; ++q)
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        float v[V];
        values<T, V>(x[q][i], v);
#pragma unroll
        for (int j = 0; j < V; ++j) mean[q] += v[j];  // (0 past D)
      }
    group_sum<A>(p.lanes, mean);
#pragma unroll
    for (int q = 0; q < A; ++q) mean[q] *= inv;
  }
#pragma unroll
  for (int q = 0; q < A; ++q) {
    rstd[q] = 0.0f;
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      if (!m.in[i]) continue;
      float v[V];
      values<T, V>(x[q][i], v);
#pragma unroll
      for (int j = 0; j < V; ++j) rstd[q] = __fmaf_rn(v[j] - mean[q], v[j] - mean[q], rstd[q]);
    }
  }
  group_sum<A>(p.lanes, rstd);
#pragma unroll
  for (int q = 0; q < A; ++q) rstd[q] = rsqrtf(__fmaf_rn(rstd[q], inv, p.eps));
}

// Heads in flight: eight fp32 elements per lane and head are 8 registers, twice.
template <typename T, int V, int kP, bool kBackward>
__host__ __device__ constexpr int at_once() {
  return V * kP * (int)sizeof(T) > 16 || kBackward ? 2 : 4;
}

// Element (token, head) row of q, k or v: [B, heads, N, D].
template <typename T>
__device__ __forceinline__ T *head_row(void *base, const RotaryParams &r, uint32_t b, uint32_t n,
                                       int64_t heads, int h) {
  return static_cast<T *>(base) + (((int64_t)b * heads + h) * r.N + n) * r.D;
}

// Heads [h0, h1) of role 0 (q), 1 (k) or 2 (v) of one token.
template <typename T, int V, int kP, bool kInterleaved>
__device__ __forceinline__ void forward_heads(const QkNormParams &p, uint32_t tok, int role, int h0,
                                              int h1) {
  constexpr int A = at_once<T, V, kP, false>();
  const RotaryParams &r = p.r;
  const bool live = tok < (uint32_t)(r.B * r.N);
  if (!live) tok = (uint32_t)(r.B * r.N) - 1;
  const uint32_t b = r.tokens.quotient(tok), n = tok - b * (uint32_t)r.N;
  Mine<V, kP> m;
  set_up<V, kP, kInterleaved, false>(p, tok, n, role < 2 && r.axes > 0, m);
  float w[kP][V], bias[kP][V], wo[kP][V], bo[kP][V];
#pragma unroll
  for (int i = 0; i < kP; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[i][j] = wo[i][j] = 1.0f;
      bias[i][j] = bo[i][j] = 0.0f;
      if (role == 2 || !m.in[i]) continue;
      const int o = kInterleaved && V > 1 ? m.e0[i] + (j ^ 1) : m.partner[i] + j;
      w[i][j] = load_as_f32(p.weight[role], p.param_dtype, m.e0[i] + j);
      wo[i][j] = load_as_f32(p.weight[role], p.param_dtype, o);
      if (p.bias[role]) {
        bias[i][j] = load_as_f32(p.bias[role], p.param_dtype, m.e0[i] + j);
        bo[i][j] = load_as_f32(p.bias[role], p.param_dtype, o);
      }
    }
  const int64_t heads = role == 0 ? r.H : r.Hk;
  const int before = role == 0 ? 0 : (int)(role == 1 ? r.H : r.H + r.Hk);
  void *const out = role == 0 ? r.q : role == 1 ? r.k : r.v;
  const T *const fused = static_cast<const T *>(r.qkv) +
                         ((int64_t)tok * (r.H + 2 * r.Hk) + before) * r.D;
  for (int h = h0; h < h1; h += A) {
    Piece<T, V> x[A][kP], o[A][kP];
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const T *row = fused + (int64_t)(h + q < h1 ? h + q : h1 - 1) * r.D;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        if (m.in[i])
          x[q][i].load(row + m.e0[i]);
        else
          zero<T, V>(x[q][i]);
        if (!kInterleaved || V == 1) {
          if (m.mask[i])
            o[q][i].load(row + m.partner[i]);
          else
            zero<T, V>(o[q][i]);
        }
      }
    }
    if (role == 2) {
#pragma unroll
      for (int q = 0; q < A; ++q)
#pragma unroll
        for (int i = 0; i < kP; ++i)
          if (live && h + q < h1 && m.in[i])
            x[q][i].store(head_row<T>(out, r, b, n, heads, h + q) + m.e0[i]);
      continue;
    }
    float mean[A], rstd[A];
    statistics<T, V, kP, A>(p, x, m, mean, rstd);
#pragma unroll
    for (int q = 0; q < A; ++q) {
      if (h + q >= h1) break;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        float v[V], u[V];
        values<T, V>(x[q][i], v);
        if (!kInterleaved || V == 1) {
          values<T, V>(o[q][i], u);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) u[j] = v[j ^ 1];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[j] = __fmaf_rn((v[j] - mean[q]) * rstd[q], w[i][j], bias[i][j]);
          u[j] = __fmaf_rn((u[j] - mean[q]) * rstd[q], wo[i][j], bo[i][j]);
          if (m.mask[i] >> j & 1) v[j] = __fmaf_rn(v[j], m.c[i][j], u[j] * m.s[i][j]);
        }
        if (live && m.in[i])
          store<T, V>(head_row<T>(out, r, b, n, heads, h + q) + m.e0[i], v);
      }
    }
  }
}

// The same heads' gradients; dw and db add up in the thread.
template <typename T, int V, int kP, bool kInterleaved>
__device__ __forceinline__ void backward_heads(const QkNormParams &p, uint32_t tok, int role,
                                               int h0, int h1, float (&dw)[kP][V],
                                               float (&db)[kP][V]) {
  constexpr int A = at_once<T, V, kP, true>();
  const RotaryParams &r = p.r;
  const bool live = tok < (uint32_t)(r.B * r.N);
  if (!live) tok = (uint32_t)(r.B * r.N) - 1;
  const uint32_t b = r.tokens.quotient(tok), n = tok - b * (uint32_t)r.N;
  Mine<V, kP> m;
  set_up<V, kP, kInterleaved, true>(p, tok, n, role < 2 && r.axes > 0, m);
  float w[kP][V];
#pragma unroll
  for (int i = 0; i < kP; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j)
      w[i][j] = role < 2 && m.in[i] ? load_as_f32(p.weight[role], p.param_dtype, m.e0[i] + j) : 0.f;
  const int64_t heads = role == 0 ? r.H : r.Hk;
  const int before = role == 0 ? 0 : (int)(role == 1 ? r.H : r.H + r.Hk);
  void *const from = role == 0 ? r.q : role == 1 ? r.k : r.v;
  const int64_t at = ((int64_t)tok * (r.H + 2 * r.Hk) + before) * r.D;
  const T *const fused = static_cast<const T *>(p.x) + at;
  T *const out = static_cast<T *>(r.qkv) + at;
  const float inv = 1.0f / (float)r.D;
  for (int h = h0; h < h1; h += A) {
    Piece<T, V> x[A][kP], g[A][kP], o[A][kP];
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const int hh = h + q < h1 ? h + q : h1 - 1;
      const T *grad = head_row<const T>(from, r, b, n, heads, hh);
      const T *row = fused + (int64_t)hh * r.D;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        zero<T, V>(x[q][i]);
        zero<T, V>(g[q][i]);
        zero<T, V>(o[q][i]);
        if (!m.in[i]) continue;
        g[q][i].load(grad + m.e0[i]);
        if (role == 2) continue;
        x[q][i].load(row + m.e0[i]);
        if ((!kInterleaved || V == 1) && m.mask[i]) o[q][i].load(grad + m.partner[i]);
      }
    }
    if (role == 2) {
#pragma unroll
      for (int q = 0; q < A; ++q)
#pragma unroll
        for (int i = 0; i < kP; ++i)
          if (live && h + q < h1 && m.in[i])
            g[q][i].store(out + (int64_t)(h + q) * r.D + m.e0[i]);
      continue;
    }
    float mean[A], rstd[A];
    statistics<T, V, kP, A>(p, x, m, mean, rstd);
    float dt[A][kP][V], sum_gn[A], sum_g[A];
#pragma unroll
    for (int q = 0; q < A; ++q) {
      sum_gn[q] = sum_g[q] = 0.0f;
      const bool counts = live && h + q < h1;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        float v[V], u[V], t[V];
        values<T, V>(x[q][i], v);
        values<T, V>(g[q][i], t);
        if (!kInterleaved || V == 1) {
          values<T, V>(o[q][i], u);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) u[j] = t[j ^ 1];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float y = m.mask[i] >> j & 1 ? __fmaf_rn(t[j], m.c[i][j], u[j] * m.s[i][j]) : t[j];
          const float norm = (v[j] - mean[q]) * rstd[q];
          dt[q][i][j] = y * w[i][j];
          if (m.in[i]) {
            sum_g[q] += dt[q][i][j];
            sum_gn[q] = __fmaf_rn(dt[q][i][j], norm, sum_gn[q]);
            if (counts) {
              dw[i][j] = __fmaf_rn(y, norm, dw[i][j]);
              db[i][j] += y;
            }
          }
        }
      }
    }
    group_sum<A>(p.lanes, sum_gn);
    if (!p.rms) group_sum<A>(p.lanes, sum_g);
#pragma unroll
    for (int q = 0; q < A; ++q) {
      if (h + q >= h1) break;
      const float a = sum_gn[q] * inv, c = p.rms ? 0.0f : sum_g[q] * inv;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        float v[V];
        values<T, V>(x[q][i], v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float norm = (v[j] - mean[q]) * rstd[q];
          v[j] = (dt[q][i][j] - c - norm * a) * rstd[q];
        }
        if (live && m.in[i]) store<T, V>(out + (int64_t)(h + q) * r.D + m.e0[i], v);
      }
    }
  }
}

__device__ __forceinline__ void unit_of(const QkNormParams &p, int u, int &role, int &h0, int &h1) {
  role = u < p.units_q ? 0 : u < p.units_qk ? 1 : 2;
  h0 = (role == 0 ? u : role == 1 ? u - p.units_q : u - p.units_qk) * p.heads_per;
  const int heads = (int)(role == 0 ? p.r.H : p.r.Hk);
  h1 = h0 + p.heads_per < heads ? h0 + p.heads_per : heads;
}

template <typename T, int V, int kP, bool kInterleaved>
__global__ void __launch_bounds__(kThreads)
    qknorm_kernel(const __grid_constant__ QkNormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  if (blockIdx.x >= p.r.turn_blocks) {
    transpose_tile<T, kP == 1 ? V : 1, false>(p.r, blockIdx.x - p.r.turn_blocks,
                                              reinterpret_cast<T *>(smem));
    return;
  }
  const uint32_t tb = blockIdx.x / (uint32_t)p.units_all;
  int role, h0, h1;
  unit_of(p, (int)(blockIdx.x - tb * (uint32_t)p.units_all), role, h0, h1);
  const uint32_t tok = tb * (kThreads / p.lanes) + threadIdx.x / p.lanes;
  forward_heads<T, V, kP, kInterleaved>(p, tok, role, h0, h1);
}

// Blocks [0, blocks_q) take q's units in turn, those up to blocks_qk k's, the rest
// v's (then v's transposed tiles, a block each).
template <typename T, int V, int kP, bool kInterleaved>
__global__ void __launch_bounds__(kThreads)
    qknorm_bwd_kernel(const __grid_constant__ QkNormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float sums[kThreads / 32][2][kMaxD];
  if (blockIdx.x >= p.blocks_all) {
    transpose_tile<T, kP == 1 ? V : 1, true>(p.r, blockIdx.x - p.blocks_all,
                                             reinterpret_cast<T *>(smem));
    return;
  }
  const int role = blockIdx.x < p.blocks_q ? 0 : blockIdx.x < p.blocks_qk ? 1 : 2;
  const uint32_t first = role == 0 ? 0 : role == 1 ? p.blocks_q : p.blocks_qk;
  const uint32_t blocks = (role == 0 ? p.blocks_q : role == 1 ? p.blocks_qk : p.blocks_all) - first;
  const int unit0 = role == 0 ? 0 : role == 1 ? p.units_q : p.units_qk;
  const uint32_t per = (role == 0 ? p.units_q : role == 1 ? p.units_qk : p.units_all) - unit0;
  float dw[kP][V], db[kP][V];
#pragma unroll
  for (int i = 0; i < kP; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
  for (uint64_t u = blockIdx.x - first; u < (uint64_t)p.token_blocks * per; u += blocks) {
    const uint32_t tb = (uint32_t)(u / per);
    int same, h0, h1;
    unit_of(p, unit0 + (int)(u - (uint64_t)tb * per), same, h0, h1);
    const uint32_t tok = tb * (kThreads / p.lanes) + threadIdx.x / p.lanes;
    backward_heads<T, V, kP, kInterleaved>(p, tok, role, h0, h1, dw, db);
  }
  if (role == 2 || !p.part) return;
  // the block's sums: over the groups of a warp, then over the warps
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < kP; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      for (int o = p.lanes; o < 32; o <<= 1) {
        dw[i][j] += __shfl_xor_sync(~0u, dw[i][j], o);
        db[i][j] += __shfl_xor_sync(~0u, db[i][j], o);
      }
      const int e = ((lane & (p.lanes - 1)) + i * p.lanes) * V + j;
      if (lane < p.lanes && e < p.r.D) {
        sums[warp][0][e] = dw[i][j];
        sums[warp][1][e] = db[i][j];
      }
    }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * p.r.D; e += kThreads) {
    const int which = e >= p.r.D, d = e - which * p.r.D;
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) t += sums[i][which][d];
    p.part[((int64_t)blockIdx.x * 2 + which) * p.r.D + d] = t;
  }
}

// Block (x, y): 32 columns of gradient y (q's weight and bias, k's weight and bias);
// eight warps take every eighth part.
struct SumArgs {
  const float *part;
  void *out[4];
  uint32_t first[4], last[4];
  int D, dtype;
};
__global__ void __launch_bounds__(kThreads) qknorm_sum_kernel(const __grid_constant__ SumArgs a) {
  __shared__ float sums[kThreads / 32][32];
  const int y = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  if (!a.out[y]) return;
  float t = 0.0f;
  if (d < a.D) {
#pragma unroll 8
    for (uint32_t i = a.first[y] + warp; i < a.last[y]; i += kThreads / 32)
      t += a.part[((int64_t)i * 2 + (y & 1)) * a.D + d];
  }
  sums[warp][lane] = t;
  __syncthreads();
  if (warp != 0 || d >= a.D) return;
  t = 0.0f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) t += sums[i][lane];
  if (a.dtype == SCMP_F32)
    static_cast<float *>(a.out[y])[d] = t;
  else if (a.dtype == SCMP_BF16)
    static_cast<__nv_bfloat16 *>(a.out[y])[d] = from_f32<__nv_bfloat16>(t);
  else
    static_cast<__half *>(a.out[y])[d] = from_f32<__half>(t);
}

int units(int64_t heads, int per) { return (int)((heads + per - 1) / per); }

template <typename T, int V, int kP, bool kInterleaved>
cudaError_t launch_p(QkNormParams p, cudaStream_t s) {
  RotaryParams &r = p.r;
  r.tokens = FastDiv((uint32_t)r.N);
  const int pieces = (r.D / V + kP - 1) / kP;
  p.lanes = 1;
  while (p.lanes < pieces) p.lanes *= 2;
  const int64_t tokens = r.B * r.N, per_block = kThreads / p.lanes;
  const int64_t token_blocks = (tokens + per_block - 1) / per_block;
  p.token_blocks = (uint32_t)token_blocks;
  // as many heads per thread as leave six units for each of the 148 SMs
  const int64_t all = r.H + r.Hk + (r.v_transposed ? 0 : r.Hk);
  const int64_t fit = all * token_blocks / (148 * 6);
  p.heads_per = (int)(fit < 1 ? 1 : fit > r.H ? r.H : fit);
  p.units_q = units(r.H, p.heads_per);
  p.units_qk = p.units_q + units(r.Hk, p.heads_per);
  p.units_all = p.units_qk + (r.v_transposed ? 0 : units(r.Hk, p.heads_per));
  const int64_t tiles = r.v_transposed ? r.B * r.Hk * ((r.N + kTile - 1) / kTile) : 0;
  const size_t smem = r.v_transposed ? (size_t)(kTile + 2) * r.D * sizeof(T) : 0;  // <= 66 KB
  int64_t blocks = token_blocks * p.units_all;
  if (r.inverse) {
    const QkNormBlocks n = qknorm_bwd_blocks(r.H, r.Hk);
    p.blocks_q = n.q;
    p.blocks_qk = n.qk;
    p.blocks_all = r.v_transposed ? n.qk : n.all;
    blocks = p.blocks_all;
  }
  if (blocks + tiles > INT32_MAX) return cudaErrorInvalidConfiguration;
  r.turn_blocks = (uint32_t)blocks;
  r.per = FastDiv((uint32_t)(r.D / V));
  auto kern = r.inverse ? qknorm_bwd_kernel<T, V, kP, kInterleaved>
                        : qknorm_kernel<T, V, kP, kInterleaved>;
  // (always the most that this kernel uses: calls at the same time agree on it)
  const int most = (kTile + 2) * kMaxD * (int)sizeof(T);
  if (most + (int)sizeof(float) * kThreads / 32 * 2 * kMaxD > 48 * 1024 && smem > 0) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
  }
  kern<<<(unsigned)(blocks + tiles), kThreads, smem, s>>>(p);
  return cudaGetLastError();
}
template <typename T, int V, int kP>
cudaError_t launch_order(const QkNormParams &p, cudaStream_t s) {
  return p.r.interleaved ? launch_p<T, V, kP, true>(p, s) : launch_p<T, V, kP, false>(p, s);
}
template <typename T, int V> bool fits(const QkNormParams &p) {
  return pieces<T, V>(p.r) && reinterpret_cast<uintptr_t>(p.x) % (V * sizeof(T)) == 0;
}
// The widest pieces (16 bytes at most) that divide every head row and half section,
// up to eight elements per lane.
template <typename T> cudaError_t launch(const QkNormParams &p, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (fits<T, 8>(p)) return launch_order<T, 8, 1>(p, s);
  if (fits<T, 4>(p))
    return p.r.D <= 128 ? launch_order<T, 4, 1>(p, s) : launch_order<T, 4, 2>(p, s);
  if (fits<T, 2>(p)) return launch_order<T, 2, 4>(p, s);
  return launch_order<T, 1, 8>(p, s);
}

}  // namespace

// Four blocks for each of the 148 SMs, shared out by heads.
QkNormBlocks qknorm_bwd_blocks(int64_t H, int64_t Hk) {
  constexpr int64_t kAll = 148 * 4;
  int64_t k = kAll * Hk / (H + 2 * Hk);
  k = k < 1 ? 1 : k;
  QkNormBlocks n;
  n.q = (uint32_t)(kAll - 2 * k);
  n.qk = n.q + (uint32_t)k;
  n.all = n.qk + (uint32_t)k;
  return n;
}

cudaError_t launch_qknorm(const QkNormParams &p, int dtype, cudaStream_t s) {
  if (dtype == SCMP_F32) return launch<float>(p, s);
  if (dtype == SCMP_BF16) return launch<__nv_bfloat16>(p, s);
  return launch<__half>(p, s);
}

cudaError_t launch_qknorm_sum(const QkNormParams &p, void *const (&grads)[4], cudaStream_t s) {
  const QkNormBlocks n = qknorm_bwd_blocks(p.r.H, p.r.Hk);
  SumArgs a;
  a.part = p.part;
  a.D = p.r.D;
  a.dtype = p.param_dtype;
  for (int y = 0; y < 4; ++y) {
    a.out[y] = grads[y];
    a.first[y] = y < 2 ? 0 : n.q;
    a.last[y] = y < 2 ? n.q : n.qk;
  }
  qknorm_sum_kernel<<<dim3((unsigned)((p.r.D + 31) / 32), 4), kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace scmp
