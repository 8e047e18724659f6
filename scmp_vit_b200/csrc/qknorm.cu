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
#include "f32x2.cuh"
#include "mx_common.cuh"
#include "qknorm.cuh"
#include "rotary_device.cuh"

namespace scmp {
namespace {

constexpr int kMaxD = 256;
// Blocks of the backward pass on an SM, by the elements of a thread.
__host__ __device__ constexpr int blocks_per_sm(int elements) { return elements > 4 ? 2 : 3; }

// A thread holds kP pieces of V elements of a head row, piece i at element (lane + i
// lanes) V of D: E = V kP values, flat, as pairs.
template <int V, int kP> struct Mine {
  static constexpr int E = V * kP;
  int e0[kP], partner[kP];
  uint32_t mask[kP];  // elements that turn
  bool in[kP];
};
template <int E> struct Pairs {
  float2 p[E / 2];
  __device__ __forceinline__ float &operator[](int e) { return reinterpret_cast<float *>(p)[e]; }
};

// Pieces, and the cos and signed sin of their elements (1 and 0 where none turns).
template <int V, int kP, bool kInterleaved, bool kBackward>
__device__ __forceinline__ void set_up(const QkNormParams &p, uint32_t tok, uint32_t n, bool turns,
                                       Mine<V, kP> &m, Pairs<V * kP> &c, Pairs<V * kP> &s) {
  const int lane = threadIdx.x & (p.lanes - 1);
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    m.e0[i] = (lane + i * p.lanes) * V;
    m.in[i] = m.e0[i] < p.r.D;
    m.mask[i] = 0;
    m.partner[i] = m.e0[i];
    float ci[V], si[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      ci[j] = 1.0f;
      si[j] = 0.0f;
    }
    if (turns && m.in[i])
      m.mask[i] = angles_of<V, kInterleaved, kBackward>(p.r, p.r.pos_batched ? tok : n, m.e0[i],
                                                        ci, si, m.partner[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      c[i * V + j] = ci[j];
      s[i * V + j] = si[j];
    }
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
template <typename T, int V, int kP>
__device__ __forceinline__ Pairs<V * kP> values(const Piece<T, V> (&x)[kP]) {
  Pairs<V * kP> r;
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    if constexpr (V == 1) {
      r[i] = to_f32(x[i].u[0]);
    } else {
      float v[V];
      x[i].get(v);
#pragma unroll
      for (int j = 0; j < V; ++j) r[i * V + j] = v[j];
    }
  }
  return r;
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
// Every element's partner within a thread's pieces (pairs side by side).
template <int E> __device__ __forceinline__ Pairs<E> swapped(const Pairs<E> &x) {
  Pairs<E> r;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) r.p[i] = make_float2(x.p[i].y, x.p[i].x);
  return r;
}

// mean and 1 / deviation of A head rows (mean 0 for rms); the variance is a second
// pass over the registers.
template <typename T, int V, int kP, int A>
__device__ __forceinline__ void statistics(const QkNormParams &p, const Piece<T, V> (&x)[A][kP],
                                           const Mine<V, kP> &m, float (&mean)[A],
                                           float (&rstd)[A]) {
  constexpr int E = V * kP;
  const float inv = 1.0f / (float)p.r.D;
#pragma unroll
  for (int q = 0; q < A; ++q) mean[q] = 0.0f;
  if (!p.rms) {
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const Pairs<E> v = values<T, V, kP>(x[q]);
      float2 t = v.p[0];
#pragma unroll
      for (int i = 1; i < E / 2; ++i) t = add2(t, v.p[i]);  // (0 past D)
      mean[q] = t.x + t.y;
    }
    group_sum<A>(p.lanes, mean);
#pragma unroll
    for (int q = 0; q < A; ++q) mean[q] *= inv;
  }
#pragma unroll
  for (int q = 0; q < A; ++q) {
    Pairs<E> v = values<T, V, kP>(x[q]);
    if (!p.rms) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) v.p[i] = add2(v.p[i], both(-mean[q]));
      if (!p.whole) {
#pragma unroll
        for (int i = 0; i < kP; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (!m.in[i]) v[i * V + j] = 0.0f;
      }
    }
    float2 t = mul2(v.p[0], v.p[0]);
#pragma unroll
    for (int i = 1; i < E / 2; ++i) t = fma2(v.p[i], v.p[i], t);
    rstd[q] = t.x + t.y;
  }
  group_sum<A>(p.lanes, rstd);
#pragma unroll
  for (int q = 0; q < A; ++q) rstd[q] = rsqrtf(__fmaf_rn(rstd[q], inv, p.eps));
}

// Heads in flight: up to 32 bytes of x per thread.
template <typename T, int V, int kP, bool kBackward>
__host__ __device__ constexpr int at_once() {
  return kBackward ? (V * kP > 4 ? 1 : 2) : V * kP * (int)sizeof(T) > 16 ? 2 : 4;
}

// Heads [h0, h1) of role 0 (q), 1 (k) or 2 (v) of one token.  With the rotation's c
// and s and the partner's weight w', an element of the output is
//   rstd (x w c + x' w' s - mean (w c + w' s)) + b c + b' s,
// whose products of weights and angles are made once per token.
template <typename T, int V, int kP, bool kInterleaved>
__device__ __forceinline__ void forward_heads(const QkNormParams &p, uint32_t tok, int role, int h0,
                                              int h1) {
  constexpr int A = at_once<T, V, kP, false>(), E = V * kP;
  constexpr bool kApart = !kInterleaved || V == 1;  // partners are other threads'
  const RotaryParams &r = p.r;
  const bool live = tok < (uint32_t)(r.B * r.N);
  if (!live) tok = (uint32_t)(r.B * r.N) - 1;
  const uint32_t b = r.tokens.quotient(tok), n = tok - b * (uint32_t)r.N;
  const int64_t heads = role == 0 ? r.H : r.Hk;
  const int before = role == 0 ? 0 : (int)(role == 1 ? r.H : r.H + r.Hk);
  const T *from = static_cast<const T *>(r.qkv) +
                  ((int64_t)tok * (r.H + 2 * r.Hk) + before + h0) * r.D;
  const int64_t apart = r.N * r.D;  // of a token's rows in q, k and v
  T *to = static_cast<T *>(role == 0 ? r.q : role == 1 ? r.k : r.v) +
          (((int64_t)b * heads + h0) * r.N + n) * r.D;
  Mine<V, kP> m;
  Pairs<E> wc, ws, shift, c, s;
  set_up<V, kP, kInterleaved, false>(p, tok, n, role < 2 && r.axes > 0, m, c, s);
  if (role < 2) {
#pragma unroll
    for (int i = 0; i < kP; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = i * V + j, at = m.e0[i] + j;
        const int o = kApart ? m.partner[i] + j : m.e0[i] + (j ^ 1);
        wc[e] = ws[e] = shift[e] = 0.0f;
        if (!m.in[i]) continue;
        wc[e] = load_as_f32(p.weight[role], p.param_dtype, at) * c[e];
        ws[e] = load_as_f32(p.weight[role], p.param_dtype, o) * s[e];
        if (p.bias[role])
          shift[e] = __fmaf_rn(load_as_f32(p.bias[role], p.param_dtype, at), c[e],
                               load_as_f32(p.bias[role], p.param_dtype, o) * s[e]);
      }
  }
  for (int h = h0; h < h1; h += A, from += A * r.D, to += A * apart) {
    Piece<T, V> x[A][kP], o[A][kP];
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const T *row = from + (h + q < h1 ? q : h1 - 1 - h) * r.D;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        if (m.in[i])
          x[q][i].load(row + m.e0[i]);
        else
          zero<T, V>(x[q][i]);
        if (kApart) {
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
          if (live && h + q < h1 && m.in[i]) x[q][i].store(to + q * apart + m.e0[i]);
      continue;
    }
    float mean[A], rstd[A];
    statistics<T, V, kP, A>(p, x, m, mean, rstd);
#pragma unroll
    for (int q = 0; q < A; ++q) {
      if (h + q >= h1) break;
      const Pairs<E> v = values<T, V, kP>(x[q]);
      Pairs<E> u, y;
      if constexpr (kApart)
        u = values<T, V, kP>(o[q]);
      else
        u = swapped<E>(v);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        float2 t = fma2(v.p[i], wc.p[i], mul2(u.p[i], ws.p[i]));
        if (!p.rms) t = fma2(both(-mean[q]), add2(wc.p[i], ws.p[i]), t);
        y.p[i] = fma2(both(rstd[q]), t, shift.p[i]);
      }
#pragma unroll
      for (int i = 0; i < kP; ++i)
        if (live && m.in[i]) store<T, V>(to + q * apart + m.e0[i], &y[i * V]);
    }
  }
}

// The same heads' gradients; dw and db add up in the thread.
template <typename T, int V, int kP, bool kInterleaved>
__device__ __forceinline__ void backward_heads(const QkNormParams &p, uint32_t tok, int role,
                                               int h0, int h1, Pairs<V * kP> &dw,
                                               Pairs<V * kP> &db) {
  constexpr int A = at_once<T, V, kP, true>(), E = V * kP;
  constexpr bool kApart = !kInterleaved || V == 1;
  const RotaryParams &r = p.r;
  const bool live = tok < (uint32_t)(r.B * r.N);
  if (!live) tok = (uint32_t)(r.B * r.N) - 1;
  const uint32_t b = r.tokens.quotient(tok), n = tok - b * (uint32_t)r.N;
  const int64_t heads = role == 0 ? r.H : r.Hk;
  const int before = role == 0 ? 0 : (int)(role == 1 ? r.H : r.H + r.Hk);
  const int64_t at = ((int64_t)tok * (r.H + 2 * r.Hk) + before + h0) * r.D;
  const T *from = static_cast<const T *>(p.x) + at;
  T *to = static_cast<T *>(r.qkv) + at;
  const int64_t apart = r.N * r.D;
  const T *grad = static_cast<const T *>(role == 0 ? r.q : role == 1 ? r.k : r.v) +
                  (((int64_t)b * heads + h0) * r.N + n) * r.D;
  Mine<V, kP> m;
  Pairs<E> c, s, w;
  set_up<V, kP, kInterleaved, true>(p, tok, n, role < 2 && r.axes > 0, m, c, s);
#pragma unroll
  for (int i = 0; i < kP; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j)
      w[i * V + j] =
          role < 2 && m.in[i] ? load_as_f32(p.weight[role], p.param_dtype, m.e0[i] + j) : 0.0f;
  const float inv = 1.0f / (float)r.D;
  for (int h = h0; h < h1; h += A, from += A * r.D, to += A * r.D, grad += A * apart) {
    Piece<T, V> x[A][kP], g[A][kP], o[A][kP];
#pragma unroll
    for (int q = 0; q < A; ++q) {
      // (what counts for no row has gradients of zero)
      const bool counts = live && h + q < h1;
      const int64_t hh = h + q < h1 ? q : h1 - 1 - h;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        zero<T, V>(x[q][i]);
        zero<T, V>(g[q][i]);
        zero<T, V>(o[q][i]);
        if (!m.in[i]) continue;
        if (counts) g[q][i].load(grad + hh * apart + m.e0[i]);
        if (role == 2) continue;
        x[q][i].load(from + hh * r.D + m.e0[i]);
        if (kApart && counts && m.mask[i]) o[q][i].load(grad + hh * apart + m.partner[i]);
      }
    }
    if (role == 2) {
#pragma unroll
      for (int q = 0; q < A; ++q)
#pragma unroll
        for (int i = 0; i < kP; ++i)
          if (live && h + q < h1 && m.in[i]) g[q][i].store(to + q * r.D + m.e0[i]);
      continue;
    }
    float mean[A], rstd[A], sum_gn[A], sum_g[A];
    statistics<T, V, kP, A>(p, x, m, mean, rstd);
    Pairs<E> norm[A], gw[A];
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const Pairs<E> v = values<T, V, kP>(x[q]), t = values<T, V, kP>(g[q]);
      Pairs<E> u;
      if constexpr (kApart)
        u = values<T, V, kP>(o[q]);
      else
        u = swapped<E>(t);
      float2 gn = make_float2(0.f, 0.f), gs = gn;
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 dt = fma2(t.p[i], c.p[i], mul2(u.p[i], s.p[i]));
        norm[q].p[i] = mul2(add2(v.p[i], both(-mean[q])), both(rstd[q]));
        gw[q].p[i] = mul2(dt, w.p[i]);  // (0 past D)
        gn = fma2(gw[q].p[i], norm[q].p[i], gn);
        gs = add2(gs, gw[q].p[i]);
        dw.p[i] = fma2(dt, norm[q].p[i], dw.p[i]);
        db.p[i] = add2(db.p[i], dt);
      }
      sum_gn[q] = gn.x + gn.y;
      sum_g[q] = gs.x + gs.y;
    }
    group_sum<A>(p.lanes, sum_gn);
    if (!p.rms) group_sum<A>(p.lanes, sum_g);
#pragma unroll
    for (int q = 0; q < A; ++q) {
      if (h + q >= h1) break;
      const float2 a = both(-sum_gn[q] * inv), d = both(p.rms ? 0.0f : -sum_g[q] * inv);
      Pairs<E> y;
#pragma unroll
      for (int i = 0; i < E / 2; ++i)
        y.p[i] = mul2(fma2(norm[q].p[i], a, add2(gw[q].p[i], d)), both(rstd[q]));
#pragma unroll
      for (int i = 0; i < kP; ++i)
        if (live && m.in[i]) store<T, V>(to + q * r.D + m.e0[i], &y[i * V]);
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
__global__ void __launch_bounds__(kThreads, blocks_per_sm(V * kP))
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
  Pairs<V * kP> dw, db;
#pragma unroll
  for (int e = 0; e < V * kP; ++e) dw[e] = db[e] = 0.0f;
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
        dw[i * V + j] += __shfl_xor_sync(~0u, dw[i * V + j], o);
        db[i * V + j] += __shfl_xor_sync(~0u, db[i * V + j], o);
      }
      const int e = ((lane & (p.lanes - 1)) + i * p.lanes) * V + j;
      if (lane < p.lanes && e < p.r.D) {
        sums[warp][0][e] = dw[i * V + j];
        sums[warp][1][e] = db[i * V + j];
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

// As many blocks as run at once on the 148 SMs, shared out by heads: of q, of q and k,
// of all.
struct Blocks {
  uint32_t q, qk, all;
};
Blocks bwd_blocks(int64_t H, int64_t Hk, int per_sm) {
  const int64_t all = 148 * per_sm;
  int64_t k = all * Hk / (H + 2 * Hk);
  k = k < 1 ? 1 : k;
  Blocks n;
  n.q = (uint32_t)(all - 2 * k);
  n.qk = n.q + (uint32_t)k;
  n.all = n.qk + (uint32_t)k;
  return n;
}

int units(int64_t heads, int per) { return (int)((heads + per - 1) / per); }

template <typename T, int V, int kP, bool kInterleaved>
cudaError_t launch_p(QkNormParams p, cudaStream_t s) {
  RotaryParams &r = p.r;
  r.tokens = FastDiv((uint32_t)r.N);
  const int pieces = (r.D / V + kP - 1) / kP;
  p.lanes = 1;
  while (p.lanes < pieces) p.lanes *= 2;
  p.whole = p.lanes * kP * V == r.D;
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
    const Blocks n = bwd_blocks(r.H, r.Hk, blocks_per_sm(V * kP));
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
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !p.part) return e;
  SumArgs a;
  a.part = p.part;
  a.D = r.D;
  a.dtype = p.param_dtype;
  for (int y = 0; y < 4; ++y) {
    a.out[y] = p.grads[y];
    a.first[y] = y < 2 ? 0 : p.blocks_q;
    a.last[y] = y < 2 ? p.blocks_q : p.blocks_qk;
  }
  qknorm_sum_kernel<<<dim3((unsigned)((r.D + 31) / 32), 4), kThreads, 0, s>>>(a);
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

size_t qknorm_part_floats(int64_t H, int64_t Hk, int64_t D) {
  return (size_t)bwd_blocks(H, Hk, blocks_per_sm(1)).qk * 2 * (size_t)D;
}

cudaError_t launch_qknorm(const QkNormParams &p, int dtype, cudaStream_t s) {
  if (dtype == SCMP_F32) return launch<float>(p, s);
  if (dtype == SCMP_BF16) return launch<__nv_bfloat16>(p, s);
  return launch<__half>(p, s);
}

}  // namespace scmp
