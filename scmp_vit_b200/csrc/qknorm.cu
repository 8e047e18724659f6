// The fused qkv projection output split into q, k and v with every head's row of q
// and k normalised and turned by multi-axis rotary positions, and its gradients.
//   n = (u - mean) / sqrt(var + eps)  or  u / sqrt(mean u^2 + eps)     over D
//   q = R(n w + b)                    R: the rotation of rotary.cu, rounded once
//   dt = R^T dq,  dw = sum dt n,  db = sum dt,  g = dt w
//   du = (g - mean(g) - n mean(g n)) / sqrt(var + eps)     (rms: without mean(g))
// Statistics are fp32 and not stored: the backward pass reads u in any case.
//
// A group of 1 to 32 lanes owns a token and walks some of its heads (a unit is a
// block's tokens by those heads): cos and sin stay in registers, a lane holds 4 or 8
// elements of a head row, sums over the row are shuffles inside the group, and a few
// heads are in flight at a time.  The partner of a pair half a section apart is loaded
// again (from L1).  Weights are kept in shared memory in fp32.  What fp32 rows are
// bound by is HBM, each element read once and written once.  16-bit rows wait for their
// loads (64 images in bf16, both directions: 41 % of HBM's rate and 48 % of the issue
// slots used, more than half of a warp's time in front of a load): two heads of 16 bytes
// per thread under way, one in the backward pass, on as many warps as registers leave.
// Sums and products go two at a time.
#include "f32x2.cuh"
#include "mx_common.cuh"
#include "qknorm.cuh"
#include "rotary_device.cuh"

namespace scmp {
namespace {

constexpr int kMaxD = 256;

// E elements of a head row per lane: x and the outputs are accessed L at a time, the
// pairs' partners (half a section apart) and the angles V at a time, V dividing L.
// Lanes hold E consecutive elements; single ones (V = 1) lie a lane apart instead.
template <typename T_, int L_, int V_, int E_, bool kInterleaved_> struct Form {
  using T = T_;
  static constexpr int L = L_, V = V_, E = E_, kLoads = E_ / L_, kPieces = E_ / V_;
  static constexpr bool kInterleaved = kInterleaved_, kApart = !kInterleaved_ || V_ == 1;
  static __device__ __forceinline__ int element(int lane, int lanes, int e) {
    return V == 1 ? lane + e * lanes : lane * E + e;
  }
};

template <int E> struct Pairs {
  float2 p[E / 2];
  __device__ __forceinline__ float &operator[](int e) { return reinterpret_cast<float *>(p)[e]; }
};

// E elements as loaded, N at a time.
template <typename T, int E, int N> struct Raw {
  Piece<T, N> u[E / N];
  __device__ __forceinline__ void zero(int i) {
    if constexpr (N == 1) {
      u[i].u[0] = from_f32<T>(0.0f);
    } else {
#pragma unroll
      for (int w = 0; w < Piece<T, N>::kWords; ++w) u[i].u[w] = 0;
    }
  }
  __device__ __forceinline__ Pairs<E> values() const {
    Pairs<E> r;
#pragma unroll
    for (int i = 0; i < E / N; ++i) {
      if constexpr (N == 1) {
        r[i] = to_f32(u[i].u[0]);
      } else {
        float v[N];
        u[i].get(v);
#pragma unroll
        for (int j = 0; j < N; ++j) r[i * N + j] = v[j];
      }
    }
    return r;
  }
  __device__ __forceinline__ void set(Pairs<E> &v) {
#pragma unroll
    for (int i = 0; i < E / N; ++i) {
      if constexpr (N == 1) {
        u[i].u[0] = from_f32<T>(v[i]);
      } else {
#pragma unroll
        for (int w = 0; w < Piece<T, N>::kWords; ++w)
          u[i].u[w] = Piece<T, N>::word(&v[i * N], w);
      }
    }
  }
};

// Every element's partner within a thread's pieces (pairs side by side).
template <int E> __device__ __forceinline__ Pairs<E> swapped(const Pairs<E> &x) {
  Pairs<E> r;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) r.p[i] = make_float2(x.p[i].y, x.p[i].x);
  return r;
}

// The section of an axis that a piece belongs to, the same for every token: kept in
// shared memory, since a thread needs it once per unit.
struct Section {
  const float2 *table;  // the piece's first cos and sin at coordinate 0
  int half, size;       // the axis's table: [size][half]
  int axis;             // -1: turned by none
  int partner;          // first element of the piece's partners
  bool second;          // of a pair's members (V = 1 or apart)
};
template <typename F>
__device__ __forceinline__ void find_sections(const QkNormParams &p, Section *sections) {
  if (threadIdx.x >= (uint32_t)p.lanes) return;
#pragma unroll 1
  for (int i = 0; i < F::kPieces; ++i) {
    const int e = F::element(threadIdx.x, p.lanes, i * F::V);
    Section s;
    s.table = p.r.table;
    s.half = s.size = 0;
    s.axis = -1;
    s.partner = e;
    s.second = false;
    int begin = 0;
#pragma unroll
    for (int a = 0; a < SCMP_MAX_AXES; ++a) {
      if (a >= p.r.axes) break;
      const int h = p.r.dims[a] >> 1, o = e - begin;
      begin += p.r.dims[a];
      if (o < 0 || e >= begin) continue;
      s.axis = a;
      s.half = h;
      s.size = p.r.sizes[a];
      s.second = F::kInterleaved ? (o & 1) : o >= h;
      s.partner = F::kInterleaved ? e ^ 1 : s.second ? e - h : e + h;
      s.table += p.r.table_at[a] + (F::kInterleaved ? o >> 1 : s.second ? o - h : o);
    }
    sections[threadIdx.x * F::kPieces + i] = s;
  }
}

// A thread's elements: first element of each load, and whether it is below D.
template <typename F> struct Lane {
  int at[F::kLoads];
  bool in[F::kLoads];
  const Section *sections;
  __device__ __forceinline__ Lane(const QkNormParams &p, const Section *all) {
    const int lane = threadIdx.x & (p.lanes - 1);
    sections = all + lane * F::kPieces;
#pragma unroll
    for (int i = 0; i < F::kLoads; ++i) {
      at[i] = F::element(lane, p.lanes, i * F::L);
      in[i] = at[i] < p.r.D;
    }
  }
};

// A group's token.
struct Token {
  uint32_t tok, b, n;
  bool live;  // (one past the last stands for that one)
  __device__ __forceinline__ Token(const QkNormParams &p, uint32_t token_block) {
    const uint32_t tokens = (uint32_t)(p.r.B * p.r.N);
    tok = token_block * (kThreads / p.lanes) + threadIdx.x / p.lanes;
    live = tok < tokens;
    if (!live) tok = tokens - 1;
    b = p.r.tokens.quotient(tok);
    n = tok - b * (uint32_t)p.r.N;
  }
};

// cos and signed sin of a thread's elements for one token (1 and 0 where nothing
// turns; a negative coordinate leaves its axis, one past the table gives NaN), and
// where each piece's partners are (-1: it does not turn).
template <typename F, bool kBackward>
__device__ __forceinline__ void angles(const QkNormParams &p, const Lane<F> &m, const Token &t,
                                       Pairs<F::E> &c, Pairs<F::E> &s,
                                       int (&partner)[F::kPieces]) {
  constexpr int V = F::V;
  constexpr bool kPaired = F::kInterleaved && V > 1;  // both members of each pair
  constexpr int N = kPaired ? V / 2 : V;
  const int64_t row = (int64_t)(p.r.pos_batched ? t.tok : t.n) * p.r.axes;
#pragma unroll
  for (int i = 0; i < F::kPieces; ++i) {
    const Section e = m.sections[i];
    const int coord = e.axis >= 0 ? __ldg(p.r.pos + row + e.axis) : -1;
    const bool turns = coord >= 0;
    partner[i] = turns ? e.partner : -1;
    float2 cs[N];
#pragma unroll
    for (int j = 0; j < N; ++j) cs[j] = make_float2(1.0f, 0.0f);
    if (turns) {
      const float2 *at = e.table + (int64_t)coord * e.half;
      const float nan = __uint_as_float(0x7FC00000u);
#pragma unroll
      for (int j = 0; j < N; ++j)
        cs[j] = coord < e.size ? __ldg(at + j) : make_float2(nan, nan);
    }
    // the first member of a pair subtracts (adds, going back)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (kPaired) {
        const int o = i * V + 2 * j;
        c[o] = c[o + 1] = cs[j].x;
        s[o] = kBackward ? cs[j].y : -cs[j].y;
        s[o + 1] = -s[o];
      } else {
        c[i * V + j] = cs[j].x;
        s[i * V + j] = e.second != kBackward ? cs[j].y : -cs[j].y;
      }
    }
  }
}

template <typename F>
__device__ __forceinline__ void load_row(const Lane<F> &m, const typename F::T *row,
                                         Raw<typename F::T, F::E, F::L> &x) {
#pragma unroll
  for (int i = 0; i < F::kLoads; ++i) {
    if (m.in[i])
      x.u[i].load(row + m.at[i]);
    else
      x.zero(i);
  }
}
template <typename F>
__device__ __forceinline__ void load_partners(const int (&partner)[F::kPieces],
                                              const typename F::T *row,
                                              Raw<typename F::T, F::E, F::V> &x) {
#pragma unroll
  for (int i = 0; i < F::kPieces; ++i) {
    if (partner[i] >= 0)
      x.u[i].load(row + partner[i]);
    else
      x.zero(i);
  }
}
template <typename F>
__device__ __forceinline__ void store_row(const Lane<F> &m, bool live, typename F::T *row,
                                          const Raw<typename F::T, F::E, F::L> &x) {
#pragma unroll
  for (int i = 0; i < F::kLoads; ++i)
    if (live && m.in[i]) x.u[i].store(row + m.at[i]);
}

// Sums over a group of lanes, of several values at a time.
template <int A> __device__ __forceinline__ void group_sum(int lanes, float (&v)[A]) {
  for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int q = 0; q < A; ++q) v[q] += __shfl_xor_sync(~0u, v[q], o);
}

// mean and 1 / deviation of A head rows (mean 0 for rms); the variance is a second
// pass over the registers.
template <typename F, int A>
__device__ __forceinline__ void statistics(const QkNormParams &p, const Lane<F> &m,
                                           const Raw<typename F::T, F::E, F::L> (&x)[A],
                                           float (&mean)[A], float (&rstd)[A]) {
  constexpr int E = F::E;
  const float inv = 1.0f / (float)p.r.D;
#pragma unroll
  for (int q = 0; q < A; ++q) mean[q] = 0.0f;
  if (!p.rms) {
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const Pairs<E> v = x[q].values();
      float2 t = v.p[0];
#pragma unroll
      for (int i = 1; i < E / 2; ++i) t = add2(t, v.p[i]);  // (0 past D)
      mean[q] = t.x + t.y;
    }
    group_sum<A>(p.lanes, mean);
#pragma unroll
    for (int q = 0; q < A; ++q) {
      // (the rounded quotient: of equal values the value itself, whatever D)
      const float m = mean[q] * inv;
      mean[q] = __fmaf_rn(__fmaf_rn(-m, (float)p.r.D, mean[q]), inv, m);
    }
  }
#pragma unroll
  for (int q = 0; q < A; ++q) {
    Pairs<E> v = x[q].values();
    if (!p.rms) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) v.p[i] = add2(v.p[i], both(-mean[q]));
      if (!p.whole) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!m.in[e / F::L]) v[e] = 0.0f;
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

// Weights and biases of q and k in shared memory, [q, k][weight, bias][kMaxD].
using Shared = float[2][2][kMaxD];  // (on 16 bytes)
__device__ __forceinline__ void load_weights(const QkNormParams &p, Shared &w) {
  for (int i = threadIdx.x; i < p.r.D; i += kThreads)
#pragma unroll
    for (int role = 0; role < 2; ++role) {
      w[role][0][i] = load_as_f32(p.weight[role], p.param_dtype, i);
      w[role][1][i] = p.bias[role] ? load_as_f32(p.bias[role], p.param_dtype, i) : 0.0f;
    }
}

// A thread's elements (kOwn), or their partners (what does not turn is its own), of
// such a row; 0 past D.
template <typename F, bool kOwn>
__device__ __forceinline__ Pairs<F::E> shared_values(const Lane<F> &m,
                                                     const int (&partner)[F::kPieces],
                                                     const float *row) {
  Pairs<F::E> r;
#pragma unroll
  for (int i = 0; i < F::kPieces; ++i) {
    const int l = i * F::V / F::L, own = m.at[l] + i * F::V % F::L;
    const int at = kOwn || !F::kApart || partner[i] < 0 ? own : partner[i];
    const bool in = m.in[l];
    if constexpr (F::V % 4 == 0) {
#pragma unroll
      for (int j = 0; j < F::V; j += 4) {
        const float4 f = in ? *reinterpret_cast<const float4 *>(row + at + j)
                            : make_float4(0.f, 0.f, 0.f, 0.f);
        r[i * F::V + j] = f.x;
        r[i * F::V + j + 1] = f.y;
        r[i * F::V + j + 2] = f.z;
        r[i * F::V + j + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < F::V; ++j) r[i * F::V + j] = in ? row[at + j] : 0.0f;
    }
  }
  if constexpr (!kOwn && !F::kApart) return swapped<F::E>(r);
  return r;
}

// What is the same for all heads of role 0 (q), 1 (k) or 2 (v): a token's rows in the
// fused tensor are D apart, in q, k and v N D.
template <typename T> struct Rows {
  T *fused, *split;
  int64_t apart;
  __device__ __forceinline__ Rows(const RotaryParams &r, void *fused_base, const Token &t,
                                  int role, int h0) {
    const int64_t heads = role == 0 ? r.H : r.Hk;
    const int64_t before = role == 0 ? 0 : role == 1 ? r.H : r.H + r.Hk;
    fused = static_cast<T *>(fused_base) + ((int64_t)t.tok * (r.H + 2 * r.Hk) + before + h0) * r.D;
    split = static_cast<T *>(role == 0 ? r.q : role == 1 ? r.k : r.v) +
            (((int64_t)t.b * heads + h0) * r.N + t.n) * r.D;
    apart = r.N * r.D;
  }
};

// Heads [h0, h1) of v, either way.
template <typename F, bool kBackward>
__device__ __forceinline__ void copy_heads(const QkNormParams &p, const Lane<F> &m,
                                           const Token &t, int h0, int h1) {
  constexpr int A = 4;
  const Rows<typename F::T> rows(p.r, p.r.qkv, t, 2, h0);
  for (int h = h0; h < h1; h += A) {
    Raw<typename F::T, F::E, F::L> x[A];
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const int64_t i = (h + q < h1 ? h + q : h1 - 1) - h0;
      load_row<F>(m, kBackward ? rows.split + i * rows.apart : rows.fused + i * p.r.D, x[q]);
    }
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const int64_t i = h + q - h0;
      if (h + q < h1)
        store_row<F>(m, t.live, kBackward ? rows.fused + i * p.r.D : rows.split + i * rows.apart,
                     x[q]);
    }
  }
}

// Heads [h0, h1) of q (role 0) or k (1).  With the partner's weight w', an element of
// the output is
//   rstd ((x - mean) w c + (x' - mean) w' s) + b c + b' s,
// whose products of weights and angles are made once per token.  The mean is taken off
// first: products with x lose what lies below the mean's last bits, a thousand times
// enlarged by the rstd of a row that is nearly constant.
template <typename F, bool kBias>
__device__ __forceinline__ void forward_heads(const QkNormParams &p, const Lane<F> &m,
                                              const Token &t, const Shared &weights, int role,
                                              int h0, int h1) {
  using T = typename F::T;
  constexpr int A = F::E > 4 ? 2 : 4, E = F::E;
  const Rows<T> rows(p.r, p.r.qkv, t, role, h0);
  const T *from = rows.fused;
  T *to = rows.split;
  Pairs<E> wc, ws, shift;
  int partner[F::kPieces];
  angles<F, false>(p, m, t, wc, ws, partner);
  if constexpr (kBias) {
    const Pairs<E> b = shared_values<F, true>(m, partner, weights[role][1]);
    const Pairs<E> o = shared_values<F, false>(m, partner, weights[role][1]);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) shift.p[i] = fma2(b.p[i], wc.p[i], mul2(o.p[i], ws.p[i]));
  }
  {
    const Pairs<E> w = shared_values<F, true>(m, partner, weights[role][0]);
    const Pairs<E> o = shared_values<F, false>(m, partner, weights[role][0]);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      wc.p[i] = mul2(w.p[i], wc.p[i]);
      ws.p[i] = mul2(o.p[i], ws.p[i]);
    }
  }
  for (int h = h0; h < h1; h += A, from += A * p.r.D, to += A * rows.apart) {
    Raw<T, E, F::L> x[A];
    Raw<T, E, F::V> o[A];
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const T *row = from + (h + q < h1 ? q : h1 - 1 - h) * p.r.D;
      load_row<F>(m, row, x[q]);
      if (F::kApart) load_partners<F>(partner, row, o[q]);
    }
    float mean[A], rstd[A];
    statistics<F, A>(p, m, x, mean, rstd);
#pragma unroll
    for (int q = 0; q < A; ++q) {
      if (h + q >= h1) break;
      Pairs<E> v = x[q].values(), u, y;
      if constexpr (F::kApart) u = o[q].values();
      if (!p.rms) {  // (what is past D or does not turn is multiplied by 0)
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          v.p[i] = add2(v.p[i], both(-mean[q]));
          if constexpr (F::kApart) u.p[i] = add2(u.p[i], both(-mean[q]));
        }
      }
      if constexpr (!F::kApart) u = swapped<E>(v);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 r = fma2(v.p[i], wc.p[i], mul2(u.p[i], ws.p[i]));
        if constexpr (kBias)
          y.p[i] = fma2(both(rstd[q]), r, shift.p[i]);
        else
          y.p[i] = mul2(both(rstd[q]), r);
      }
      x[q].set(y);
      store_row<F>(m, t.live, to + q * rows.apart, x[q]);
    }
  }
}

// The same heads' gradients; dw and db add up in the thread, and over its units in
// shared memory: sums holds E (with biases 2 E) values, a thread's kThreads apart.
template <typename F, bool kBias>
__device__ __forceinline__ void backward_heads(const QkNormParams &p, const Lane<F> &m,
                                               const Token &t, const Shared &weights,
                                               const Pairs<F::E> &c, const Pairs<F::E> &s,
                                               const int (&partner)[F::kPieces], int role, int h0,
                                               int h1, float *sums) {
  using T = typename F::T;
  constexpr int A = F::E > 4 ? 1 : 2, E = F::E;
  const Rows<T> rows(p.r, p.r.qkv, t, role, h0);
  const T *from = static_cast<const T *>(p.x) + (rows.fused - static_cast<T *>(p.r.qkv));
  T *to = rows.fused;
  const T *grad = rows.split;
  const float inv = 1.0f / (float)p.r.D;
  Pairs<E> dw, db;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) dw.p[i] = db.p[i] = make_float2(0.f, 0.f);
  for (int h = h0; h < h1; h += A, from += A * p.r.D, to += A * p.r.D, grad += A * rows.apart) {
    Raw<T, E, F::L> x[A], g[A];
    Raw<T, E, F::V> o[A];
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const int64_t i = h + q < h1 ? q : h1 - 1 - h;
      load_row<F>(m, from + i * p.r.D, x[q]);
      if (t.live && h + q < h1) {
        load_row<F>(m, grad + i * rows.apart, g[q]);
        if (F::kApart) load_partners<F>(partner, grad + i * rows.apart, o[q]);
      } else {  // (what counts for no row has gradients of zero)
#pragma unroll
        for (int l = 0; l < F::kLoads; ++l) g[q].zero(l);
#pragma unroll
        for (int l = 0; l < F::kPieces; ++l) o[q].zero(l);
      }
    }
    float mean[A], rstd[A], sum_gn[A], sum_g[A];
    statistics<F, A>(p, m, x, mean, rstd);
    Pairs<E> norm[A], gw[A];
    const Pairs<E> w = shared_values<F, true>(m, partner, weights[role][0]);
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const Pairs<E> v = x[q].values(), y = g[q].values();
      Pairs<E> u;
      if constexpr (F::kApart)
        u = o[q].values();
      else
        u = swapped<E>(y);
      float2 gn = make_float2(0.f, 0.f), gs = gn;
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 dt = fma2(y.p[i], c.p[i], mul2(u.p[i], s.p[i]));
        norm[q].p[i] = mul2(add2(v.p[i], both(-mean[q])), both(rstd[q]));
        gw[q].p[i] = mul2(dt, w.p[i]);  // (0 past D)
        gn = fma2(gw[q].p[i], norm[q].p[i], gn);
        gs = add2(gs, gw[q].p[i]);
        dw.p[i] = fma2(dt, norm[q].p[i], dw.p[i]);
        if (kBias) db.p[i] = add2(db.p[i], dt);
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
      x[q].set(y);
      store_row<F>(m, t.live, to + q * p.r.D, x[q]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    sums[e * kThreads] += dw[e];
    if (kBias) sums[(E + e) * kThreads] += db[e];
  }
}

// A unit's heads among q's, k's and v's in a row: f(role, first, last).
template <typename Fn>
__device__ __forceinline__ void for_roles(const QkNormParams &p, uint32_t split, Fn &&f) {
  const int H = (int)p.r.H, Hk = (int)p.r.Hk, all = H + Hk + (p.r.v_transposed ? 0 : Hk);
  const int first = (int)split * p.heads_per;
  const int last = first + p.heads_per < all ? first + p.heads_per : all;
  if (first < H) f(0, first, last < H ? last : H);
  if (last > H && first < H + Hk)
    f(1, first > H ? first - H : 0, last < H + Hk ? last - H : Hk);
  if (last > H + Hk) f(2, first > H + Hk ? first - H - Hk : 0, last - H - Hk);
}

// Blocks take units in turn (behind them v's transposed tiles, a block each).
// (the narrower the pieces, the more registers their places take)
template <typename F, bool kBackward> __host__ __device__ constexpr int blocks_per_sm() {
  return F::V <= 2 || (kBackward && F::E > 4 && sizeof(typename F::T) == 4) ? 2 : 3;
}
template <typename F, bool kBias>
__global__ void __launch_bounds__(kThreads, (blocks_per_sm<F, false>()))
    qknorm_kernel(const __grid_constant__ QkNormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) Shared weights;
  if (blockIdx.x >= p.r.turn_blocks) {
    transpose_tile<typename F::T, F::L, false>(p.r, blockIdx.x - p.r.turn_blocks,
                                               reinterpret_cast<typename F::T *>(smem));
    return;
  }
  __shared__ Section sections[32 * F::kPieces];
  load_weights(p, weights);
  find_sections<F>(p, sections);
  const Lane<F> m(p, sections);
  __syncthreads();
  for (uint32_t u = blockIdx.x; u < p.units; u += p.r.turn_blocks) {
    const uint32_t tb = u / p.splits;
    const Token t(p, tb);
    for_roles(p, u - tb * p.splits, [&](int role, int h0, int h1) {
      if (role == 2)
        copy_heads<F, false>(p, m, t, h0, h1);
      else
        forward_heads<F, kBias>(p, m, t, weights, role, h0, h1);
    });
  }
}


template <typename F, bool kBias>
__global__ void __launch_bounds__(kThreads, (blocks_per_sm<F, true>()))
    qknorm_bwd_kernel(const __grid_constant__ QkNormParams p) {
  constexpr int E = F::E;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) Shared weights;
  __shared__ Section sections[32 * F::kPieces];
  // [q, k][weight, bias][E][kThreads], a column per thread; then [warps][kMaxD] for one
  constexpr int kKinds = kBias ? 2 : 1;
  __shared__ float sums[2 * kKinds * E * kThreads];
  if (blockIdx.x >= p.r.turn_blocks) {
    transpose_tile<typename F::T, F::L, true>(p.r, blockIdx.x - p.r.turn_blocks,
                                              reinterpret_cast<typename F::T *>(smem));
    return;
  }
  load_weights(p, weights);
  find_sections<F>(p, sections);
  float *const mine = sums + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2 * kKinds * E; ++i) mine[i * kThreads] = 0.0f;
  const Lane<F> m(p, sections);
  __syncthreads();
  for (uint32_t u = blockIdx.x; u < p.units; u += p.r.turn_blocks) {
    const uint32_t tb = u / p.splits;
    const Token t(p, tb);
    Pairs<E> c, s;
    int partner[F::kPieces];
    angles<F, true>(p, m, t, c, s, partner);
    for_roles(p, u - tb * p.splits, [&](int role, int h0, int h1) {
      if (role == 2)
        copy_heads<F, true>(p, m, t, h0, h1);
      else
        backward_heads<F, kBias>(p, m, t, weights, c, s, partner, role, h0, h1,
                                 mine + role * kKinds * E * kThreads);
    });
  }
  if (!p.part) return;
  // the block's sums: over the groups of a warp, then over the warps, one gradient
  // after the other (its thread columns are read before they are written over)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 1
  for (int k = 0; k < 2 * kKinds; ++k) {
    float *const part = sums + k * E * kThreads;  // [warps][kMaxD] fits: 32 E >= lanes E
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = mine[(k * E + e) * kThreads];
      for (int o = p.lanes; o < 32; o <<= 1) v[e] += __shfl_xor_sync(~0u, v[e], o);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane < p.lanes) part[warp * 32 * E + F::element(lane, p.lanes, e)] = v[e];
    __syncthreads();
    const int role = k / kKinds, which = k % kKinds;
    for (int d = threadIdx.x; d < p.r.D; d += kThreads) {
      float t = 0.0f;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) t += part[i * 32 * E + d];
      p.part[(((int64_t)blockIdx.x * 2 + role) * 2 + which) * p.r.D + d] = t;
    }
  }
}

// Block (x, y): 32 columns of gradient y (q's weight and bias, k's weight and bias);
// 32 warps take every 32nd part.
struct SumArgs {
  const float *part;
  void *out[4];
  uint32_t parts;
  int D, dtype;
};
__global__ void __launch_bounds__(1024) qknorm_sum_kernel(const __grid_constant__ SumArgs a) {
  __shared__ float sums[32][33];
  const int y = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  if (!a.out[y]) return;
  float t = 0.0f;
  if (d < a.D) {
#pragma unroll 8
    for (uint32_t i = warp; i < a.parts; i += 32) t += a.part[((int64_t)i * 4 + y) * a.D + d];
  }
  sums[warp][lane] = t;
  __syncthreads();
  t = sums[lane][warp];  // column `warp` of the block, its parts over the lanes
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
  const int c = blockIdx.x * 32 + warp;
  if (lane != 0 || c >= a.D) return;
  if (a.dtype == SCMP_F32)
    static_cast<float *>(a.out[y])[c] = t;
  else if (a.dtype == SCMP_BF16)
    static_cast<__nv_bfloat16 *>(a.out[y])[c] = from_f32<__nv_bfloat16>(t);
  else
    static_cast<__half *>(a.out[y])[c] = from_f32<__half>(t);
}

template <typename F> cudaError_t launch_form(QkNormParams p, cudaStream_t s) {
  using T = typename F::T;
  RotaryParams &r = p.r;
  r.tokens = FastDiv((uint32_t)r.N);
  p.lanes = 1;
  while (p.lanes * F::E < r.D) p.lanes *= 2;
  p.whole = p.lanes * F::E == r.D;
  const int64_t tokens = r.B * r.N, per_block = kThreads / p.lanes;
  const int64_t token_blocks = (tokens + per_block - 1) / per_block;
  // as many heads per unit as leave 24 units for each of the 148 SMs, so that the last
  // ones to run are a small part (12: 8 clips forward 36 us instead of 34); 8 where
  // elements go one at a time, whose angles cost a unit more than its heads do (odd half
  // sections, bf16 [32, 257], 24 heads of 128: 87 + 119 us, with 24 units 122 + 152)
  const int64_t all = r.H + r.Hk + (r.v_transposed ? 0 : r.Hk);
  int64_t splits = (148 * (F::V == 1 ? 8 : 24) + token_blocks - 1) / token_blocks;
  splits = splits > all ? all : splits;
  p.heads_per = (int)((all + splits - 1) / splits);
  p.splits = (uint32_t)((all + p.heads_per - 1) / p.heads_per);
  const int64_t tiles = r.v_transposed ? r.B * r.Hk * ((r.N + kTile - 1) / kTile) : 0;
  const size_t smem = r.v_transposed ? (size_t)(kTile + 2) * r.D * sizeof(T) : 0;  // <= 66 KB
  const int64_t units = token_blocks * p.splits;
  if (units + tiles > INT32_MAX) return cudaErrorInvalidConfiguration;
  p.units = (uint32_t)units;
  const uint32_t most = 148u * (r.inverse ? blocks_per_sm<F, true>() : blocks_per_sm<F, false>());
  r.turn_blocks = p.units < most ? p.units : most;
  const bool bias = r.inverse ? p.grads[1] || p.grads[3] : p.bias[0] || p.bias[1];
  auto kern = r.inverse ? (bias ? qknorm_bwd_kernel<F, true> : qknorm_bwd_kernel<F, false>)
                        : (bias ? qknorm_kernel<F, true> : qknorm_kernel<F, false>);
  if (smem > 0) {
    // (always the most that this kernel uses: calls at the same time agree on it)
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (kTile + 2) * kMaxD * (int)sizeof(T));
    if (e != cudaSuccess) return e;
  }
  kern<<<(unsigned)(r.turn_blocks + tiles), kThreads, smem, s>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !p.part) return e;
  SumArgs a;
  a.part = p.part;
  a.parts = r.turn_blocks;
  a.D = r.D;
  a.dtype = p.param_dtype;
  for (int y = 0; y < 4; ++y) a.out[y] = p.grads[y];
  qknorm_sum_kernel<<<dim3((unsigned)((r.D + 31) / 32), 4), 1024, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T, int L, int V, int E>
cudaError_t launch_order(const QkNormParams &p, cudaStream_t s) {
  return p.r.interleaved ? launch_form<Form<T, L, V, E, true>>(p, s)
                         : launch_form<Form<T, L, V, E, false>>(p, s);
}
// Whether rows can be accessed L elements at a time, and pairs V.
template <typename T, int L, int V> bool fits(const QkNormParams &p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.r.qkv) | reinterpret_cast<uintptr_t>(p.r.q) |
                       reinterpret_cast<uintptr_t>(p.r.k) | reinterpret_cast<uintptr_t>(p.r.v) |
                       reinterpret_cast<uintptr_t>(p.x);
  bool ok = p.r.D % L == 0 && at % (L * sizeof(T)) == 0;
  // (a piece lies in one section, and in one half of it where pairs are apart)
  for (int a = 0; a < p.r.axes; ++a)
    ok = ok && p.r.dims[a] / (p.r.interleaved ? 1 : 2) % V == 0;
  return ok;
}
// The widest accesses (16 bytes at most) that rows and half sections allow.  Eight
// elements per lane; four of fp32 in the forward pass where 32 lanes hold the row so
// (64 images of 16 heads of 64: 72 us, with eight 75; backward 131 and 120).
template <typename T> cudaError_t launch(const QkNormParams &p, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (fits<T, 8, 8>(p)) return launch_order<T, 8, 8, 8>(p, s);
    if (fits<T, 8, 4>(p)) return launch_order<T, 8, 4, 8>(p, s);
    if (fits<T, 4, 4>(p)) return launch_order<T, 4, 4, 8>(p, s);
  } else {
    if (fits<T, 4, 4>(p))
      return p.r.D <= 128 && !p.r.inverse ? launch_order<T, 4, 4, 4>(p, s)
                                          : launch_order<T, 4, 4, 8>(p, s);
  }
  if (fits<T, 2, 2>(p)) return launch_order<T, 2, 2, 8>(p, s);
  return launch_order<T, 1, 1, 8>(p, s);
}

}  // namespace

size_t qknorm_part_floats(int64_t D) {
  return (size_t)148 * blocks_per_sm<Form<float, 4, 4, 4, true>, true>() * 4 * (size_t)D;
}

cudaError_t launch_qknorm(const QkNormParams &p, int dtype, cudaStream_t s) {
  if (dtype == SCMP_F32) return launch<float>(p, s);
  if (dtype == SCMP_BF16) return launch<__nv_bfloat16>(p, s);
  return launch<__half>(p, s);
}

}  // namespace scmp
