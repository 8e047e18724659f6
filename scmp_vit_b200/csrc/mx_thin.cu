// The 4-bit product for a few activation rows (single tokens): bound by one read
// of the weight and by latency, so one launch does everything.
//
// Every block quantises the rows itself (or widens their codes) into shared
// memory, as fp16 values and fp32 scales, while its first weight rows are on
// their way.  A warp takes an output feature: 16 bytes of weight per lane are 32
// codes, i.e. a block of 32 (mxfp4) or two of 16 (nvfp4).  Products of e2m1
// values are multiples of 1/4 up to 36: eight of them add up exactly in fp16,
// which the four accumulators per block rely on; block sums and scales are fp32.
// One row, [4096, 1024]: 4.3 us with the weight from HBM, 3.6 from L2 (quantise +
// tensor-core tiles 6.7 and 6.0); mx_thin has the sizes where it pays.
#include "mx_common.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 2;  // 1024-value steps of a weight row in flight

__device__ __forceinline__ void store_as(void *p, int dtype, int64_t i, float v) {
  if (dtype == SCMP_F32)
    static_cast<float *>(p)[i] = v;
  else if (dtype == SCMP_BF16)
    static_cast<__nv_bfloat16 *>(p)[i] = from_f32<__nv_bfloat16>(v);
  else
    static_cast<__half *>(p)[i] = from_f32<__half>(v);
}

// Eight codes to eight fp16 values.
__device__ __forceinline__ uint4 widen8(uint32_t codes) {
  uint4 r;
  asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}\n"
      : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
      : "r"(codes));
  return r;
}
template <int kFmt> __device__ __forceinline__ float scale_value(uint32_t code) {
  if (kFmt == SCMP_NVFP4) return e4m3_value(code);
  return code == kMxNan ? __uint_as_float(0x7FC00000u) : e8m0_value(code);
}
__device__ __forceinline__ __half2 as_half2(uint32_t w) {
  return *reinterpret_cast<const __half2 *>(&w);
}
// Smaller and larger of two scales, a NaN if either is one.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Sum of eight products, exact in fp16 until the two halves meet in fp32.
__device__ __forceinline__ float dot8(const uint4 &w, const uint4 &x) {
  __half2 a = __hmul2(as_half2(w.x), as_half2(x.x));
  a = __hfma2(as_half2(w.y), as_half2(x.y), a);
  a = __hfma2(as_half2(w.z), as_half2(x.z), a);
  a = __hfma2(as_half2(w.w), as_half2(x.w), a);
  const float2 f = __half22float2(a);
  return f.x + f.y;
}

// The 16 bytes of 32 codes and their scales (two 16-value blocks of nvfp4).
template <int kFmt> struct Step {
  uint4 codes;
  float s0, s1;
  __device__ __forceinline__ void load(const MxProduct &p, int64_t n, int64_t k, int64_t kp,
                                       int64_t groups) {
    codes = make_uint4(0, 0, 0, 0);
    s0 = s1 = 0.0f;
    if (k >= kp) return;
    codes = __ldg(reinterpret_cast<const uint4 *>(p.b + n * (kp >> 1) + (k >> 1)));
    const int64_t b = k / (kFmt == SCMP_MXFP4 ? 32 : 16);
    const uint8_t *at = p.b_scales + mx_scale_word(n, b >> 2, groups) + (b & 3);
    s0 = scale_value<kFmt>(__ldg(at));
    if (kFmt == SCMP_NVFP4) s1 = scale_value<kFmt>(__ldg(at + 1));  // b is even: same word
  }
};

// Rows of x (T, or their codes when kCodes) to shared memory: scales [M][kp /
// block] fp32 and values [M][kp] fp16, the four 16-byte pieces of 32 values a
// quarter row apart, so that the lanes' reads (32 values each) are neighbours.
template <typename T, int kFmt, bool kCodes>
__device__ __forceinline__ void stage_rows(const MxProduct &p, const T *x, int64_t ld, int M,
                                           int64_t kp, int64_t groups, bool vec, uint4 *values,
                                           float *scales) {
  constexpr int kLanes = kFmt == SCMP_MXFP4 ? 4 : 2;  // lanes per block, 8 values each
  constexpr int kAtOnce = 2;                          // pieces of 8 values per thread
  const int pieces = (int)(kp >> 3), blocks = pieces / kLanes, total = M * pieces;
  // (whole warps take part: the lanes of a block meet in shuffles)
  for (int i0 = threadIdx.x; i0 - (int)(threadIdx.x & 31) < total; i0 += kThreads * kAtOnce) {
    float v[kAtOnce][8];
    uint32_t codes[kAtOnce], scale[kAtOnce];
    int m[kAtOnce], q[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = i0 + j * kThreads;
      m[j] = i / pieces;
      q[j] = i - m[j] * pieces;  // piece of the row
      codes[j] = scale[j] = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t) v[j][t] = 0.0f;
      if (i >= total) continue;
      if (kCodes) {
        codes[j] = __ldg(reinterpret_cast<const uint32_t *>(p.a + m[j] * (kp >> 1)) + q[j]);
        const int b = q[j] / kLanes;
        scale[j] = __ldg(p.a_scales + mx_scale_word(m[j], b >> 2, groups) + (b & 3));
      } else {
        const T *src = x + m[j] * ld + q[j] * 8;
        if (vec && q[j] * 8 + 8 <= p.K) {
#pragma unroll
          for (int t = 0; t < 8; t += kVec16<T>)
            unpack16<T>(__ldg(reinterpret_cast<const uint4 *>(src + t)), v[j] + t);
        } else {
#pragma unroll
          for (int t = 0; t < 8; ++t)
            if (q[j] * 8 + t < p.K) v[j][t] = to_f32(src[t]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (!kCodes) {
        uint32_t amax = max_bits<8>(v[j]);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) amax = max(amax, __shfl_xor_sync(~0u, amax, o));
        scale[j] = mx_encode8<kFmt, false>(v[j], amax, 1.0f, &codes[j]);
      }
      if (i0 + j * kThreads < total) {
        values[m[j] * pieces + (q[j] & 3) * (pieces >> 2) + (q[j] >> 2)] = widen8(codes[j]);
        if ((q[j] & (kLanes - 1)) == 0)
          scales[m[j] * blocks + q[j] / kLanes] = scale_value<kFmt>(scale[j]);
      }
    }
  }
}

template <typename T, int kFmt, bool kCodes, int kM>
__global__ void __launch_bounds__(kThreads)
    mx_thin_kernel(const __grid_constant__ MxProduct p, const T *__restrict__ x, int64_t ld,
                   int64_t kp, int64_t groups, bool vec) {
  extern __shared__ __align__(16) uint4 smem[];
  constexpr int kBlock = kFmt == SCMP_MXFP4 ? 32 : 16;
  const int M = (int)p.M, pieces = (int)(kp >> 3), blocks = (int)(kp / kBlock);
  float *scales = reinterpret_cast<float *>(smem + (size_t)M * pieces);
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  int64_t n = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);

  Step<kFmt> w[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (n < p.N) w[i].load(p, n, i * 1024 + lane * 32, kp, groups);
  stage_rows<T, kFmt, kCodes>(p, x, ld, M, kp, groups, vec, smem, scales);
  __syncthreads();
  for (; n < p.N; n += warps) {
    float acc[kM];
#pragma unroll
    for (int m = 0; m < kM; ++m) acc[m] = 0.0f;
    for (int64_t k0 = 0; k0 < kp; k0 += kAhead * 1024) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t k = k0 + i * 1024 + lane * 32;
        const Step<kFmt> s = w[i];
        // this slot's next piece: further along the row, or of the next row
        if (k0 + kAhead * 1024 < kp)
          w[i].load(p, n, k + kAhead * 1024, kp, groups);
        else if (n + warps < p.N)
          w[i].load(p, n + warps, i * 1024 + lane * 32, kp, groups);
        if (k >= kp) continue;
        const uint4 c[4] = {widen8(s.codes.x), widen8(s.codes.y), widen8(s.codes.z),
                            widen8(s.codes.w)};
#pragma unroll
        for (int m = 0; m < kM; ++m) {
          if (m >= M) break;
          const int quarter = pieces >> 2;
          const uint4 *v = smem + m * pieces + (k >> 5);
          const float *sx = scales + m * blocks + k / kBlock;
          const float lo = dot8(c[0], v[0]) + dot8(c[1], v[quarter]);
          const float hi = dot8(c[2], v[2 * quarter]) + dot8(c[3], v[3 * quarter]);
          if (kFmt == SCMP_MXFP4)  // the smaller scale first: nothing leaves fp32's range on the way
            acc[m] = __fmaf_rn((lo + hi) * min_nan(s.s0, sx[0]), max_nan(s.s0, sx[0]), acc[m]);
          else
            acc[m] = __fmaf_rn(lo * s.s0, sx[0], __fmaf_rn(hi * s.s1, sx[1], acc[m]));
        }
      }
    }
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      if (m >= M) break;
      float v = acc[m];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
      if (lane == 0) {
        const float bias = p.bias ? load_as_f32(p.bias, p.bias_dtype, n) : 0.0f;
        store_as(p.out, p.out_dtype, m * p.N + n, __fmaf_rn(v, p.alpha, bias));
      }
    }
  }
}

template <typename T, int kFmt, bool kCodes, int kM>
cudaError_t launch(const MxProduct &p, const void *x, int64_t ld, const MxLayout &l,
                   cudaStream_t s) {
  auto kern = mx_thin_kernel<T, kFmt, kCodes, kM>;
  const size_t smem = (size_t)p.M * l.kp * 2 + (size_t)p.M * (l.kp / l.block) * 4;
  if (smem > 48 * 1024) {
    // (always the most that this kernel uses: calls at the same time agree on it)
    const cudaError_t e = cudaFuncSetAttribute(
        kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
        kM * (SCMP_MX_THIN_K * 2 + SCMP_MX_THIN_K / (kFmt == SCMP_MXFP4 ? 32 : 16) * 4));
    if (e != cudaSuccess) return e;
  }
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld * (int)sizeof(T) % 16 == 0;
  // eight blocks on each of the 148 SMs for one row; more rows cost more to
  // stage, so fewer blocks stage them (four rows, [4096, 1024]: 6.1 against 7.5 us)
  const int64_t blocks = (p.N + kThreads / 32 - 1) / (kThreads / 32);
  const int64_t most = 148 * (kM == 1 ? 8 : 2);
  kern<<<(unsigned)(blocks < most ? blocks : most), kThreads, smem, s>>>(
      p, static_cast<const T *>(x), ld, l.kp, l.groups, vec);
  return cudaGetLastError();
}
template <typename T, int kFmt, bool kCodes>
cudaError_t launch_m(const MxProduct &p, const void *x, int64_t ld, const MxLayout &l,
                     cudaStream_t s) {
  if (p.M == 1) return launch<T, kFmt, kCodes, 1>(p, x, ld, l, s);
  if (p.M == 2) return launch<T, kFmt, kCodes, 2>(p, x, ld, l, s);
  return launch<T, kFmt, kCodes, SCMP_MX_THIN_ROWS>(p, x, ld, l, s);
}
template <int kFmt>
cudaError_t launch_f(const MxProduct &p, const void *x, int x_dtype, int64_t ld, const MxLayout &l,
                     cudaStream_t s) {
  if (!x) return launch_m<float, kFmt, true>(p, nullptr, 0, l, s);
  if (x_dtype == SCMP_F32) return launch_m<float, kFmt, false>(p, x, ld, l, s);
  if (x_dtype == SCMP_BF16) return launch_m<__nv_bfloat16, kFmt, false>(p, x, ld, l, s);
  return launch_m<__half, kFmt, false>(p, x, ld, l, s);
}

}  // namespace

bool mx_thin_fits(int64_t M, int64_t K) { return M <= SCMP_MX_THIN_ROWS && K <= SCMP_MX_THIN_K; }

// With k = K / 1024 and n = N / 1024 this launch takes about 2 + k n (0.25 +
// 0.17 M) + 0.25 M k us, quantise + tensor-core tiles 4.6 + 1.25 k.  mxfp4, [N, K]
// and rows, this / the other (us, weights from HBM):
//   [1024, 1024]  1: 2.6 / 6.0   4: 3.8 / 6.0     [4096, 1024]  1: 4.3 / 6.7   4: 6.9 / 6.7
//   [1024, 4096]  1: 5.7 / 9.8   4: 9.6 / 9.8     [4096, 4096]  1: 7.5 / 10.0  2: 11.6 / 10.0
//   [16384, 1024] 1: 9.1 / 7.4                    [6144, 6144]  1: 15.0 / 12.2
bool mx_thin(int64_t M, int64_t N, int64_t K) {
  return mx_thin_fits(M, K) &&
         K / 1024.0 * (N / 1024.0 * (1 + 0.7 * M) + (double)M - 5) < 12;
}

cudaError_t launch_mx_thin(const MxProduct &p, const void *x, int x_dtype, int64_t ld,
                           cudaStream_t s) {
  const MxLayout l = mx_layout(p.M, p.K, p.fmt);
  return p.fmt == SCMP_MXFP4 ? launch_f<SCMP_MXFP4>(p, x, x_dtype, ld, l, s)
                             : launch_f<SCMP_NVFP4>(p, x, x_dtype, ld, l, s);
}

}  // namespace scmp
