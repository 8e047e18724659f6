// The 8-bit product for a few rows (single tokens): bound by one read of the
// weight and by latency, so one launch does everything.
//
// Every block quantises the rows itself (or widens their codes) into shared
// memory, as fp32 values of the codes, while its first weight rows are on their
// way.  A warp takes an output feature: 16 bytes of weight per lane are 16 codes,
// an eighth of a block.  Products of two e4m3 values are exact in fp32; 16 of them
// are summed, then scaled by the two blocks' powers of two and added up in fp32.
#include "fp8_common.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 2;  // steps of a weight row in flight (four: [4096, 4096] 9.3 -> 10.5 us)
constexpr int kStepValues = 512;  // values of a warp's step

__device__ __forceinline__ void store_as(void *p, int dtype, int64_t i, float v) {
  if (dtype == SCMP_F32)
    static_cast<float *>(p)[i] = v;
  else if (dtype == SCMP_BF16)
    static_cast<__nv_bfloat16 *>(p)[i] = from_f32<__nv_bfloat16>(v);
  else
    static_cast<__half *>(p)[i] = from_f32<__half>(v);
}

// acc + sum 2^(a + b - 254) for two scale codes.  The power is one normal number
// except near the ends of fp32's range, where it goes in two factors.
__device__ __forceinline__ float add_scaled(float acc, float sum, uint32_t a, uint32_t b) {
  const int field = (int)(a + b) - 127;  // exponent field of the product
  if (a != kFp8Nan && b != kFp8Nan && field >= 1 && field <= 254)
    return __fmaf_rn(sum, __uint_as_float((uint32_t)field << 23), acc);
  if (a == kFp8Nan || b == kFp8Nan) return __uint_as_float(0x7FC00000u);
  const int one = field < 1 ? 1 : 254;
  int rest = field - one + 127;
  rest = rest < 0 ? 0 : rest;  // (below every fp32 number)
  return __fmaf_rn(sum * __uint_as_float((uint32_t)one << 23),
                   __uint_as_float((uint32_t)rest << 23), acc);
}

struct Step {
  uint4 codes;
  uint32_t scale;
  __device__ __forceinline__ void load(const Fp8Product &p, int64_t n, int64_t k,
                                       const Fp8Layout &l) {
    codes = make_uint4(0, 0, 0, 0);
    scale = 0;
    if (k >= l.kp) return;
    codes = __ldg(reinterpret_cast<const uint4 *>(p.b + n * l.kp + k));
    scale = __ldg(p.b_scales + fp8_scale_at(n, k / kFp8Block, l.groups));
  }
};

// Rows of x (T, or their codes when kCodes) to shared memory: scale codes [M]
// [blocks] and the codes' values [M][pieces of 16 values], the four 16-byte parts
// of a piece a quarter of the row apart, so that the lanes' reads (a piece each)
// are neighbours.
template <typename T, bool kCodes>
__device__ __forceinline__ void stage_rows(const Fp8Product &p, const T *x, int64_t ld, int M,
                                           const Fp8Layout &l, bool vec, float4 *values,
                                           uint32_t *scales) {
  const int pieces = (int)(l.kp >> 4), eighths = (int)l.blocks * 16, total = M * eighths;
  // 8 values per thread, 16 lanes per block (whole warps take part)
  for (int i = threadIdx.x; i - (int)(threadIdx.x & 31) < total; i += kThreads) {
    const int m = i / eighths, q = i - m * eighths;  // eighth of a block's lane: values 8 q ..
    float v[8];
    uint32_t scale = 0;
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = 0.0f;
    const bool live = i < total;
    if (live) {
      if (kCodes) {
        if (q * 8 < l.kp) {
          const uint2 c = __ldg(reinterpret_cast<const uint2 *>(p.a + m * l.kp + q * 8));
          e4m3_values(c.x, v);
          e4m3_values(c.y, v + 4);
        }
        scale = __ldg(p.a_scales + fp8_scale_at(m, q >> 4, l.groups));
      } else {
        const T *src = x + m * ld + q * 8;
        if (vec && q * 8 + 8 <= p.K) {
#pragma unroll
          for (int t = 0; t < 8; t += kVec16<T>)
            unpack16<T>(__ldg(reinterpret_cast<const uint4 *>(src + t)), v + t);
        } else {
#pragma unroll
          for (int t = 0; t < 8; ++t)
            if (q * 8 + t < p.K) v[t] = to_f32(src[t]);
        }
      }
    }
    if (!kCodes) {
      uint32_t amax = max_bits<8>(v);
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) amax = max(amax, __shfl_xor_sync(~0u, amax, o));
      scale = fp8_scale(amax);
      const float inv = fp8_inverse(scale);
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] *= inv;
      e4m3_values(e4m3x4(v[0], v[1], v[2], v[3]), v);
      e4m3_values(e4m3x4(v[4], v[5], v[6], v[7]), v + 4);
    }
    if (live && q * 8 < l.kp) {
      float4 *at = values + m * pieces * 4 + (q & 1) * 2 * pieces + (q >> 1);
      at[0] = make_float4(v[0], v[1], v[2], v[3]);
      at[pieces] = make_float4(v[4], v[5], v[6], v[7]);
    }
    if (live && (q & 15) == 0) scales[m * (int)l.blocks + (q >> 4)] = scale;
  }
}

template <typename T, bool kCodes, int kM>
__global__ void __launch_bounds__(kThreads)
    fp8_thin_kernel(const __grid_constant__ Fp8Product p, const T *__restrict__ x, int64_t ld,
                    const __grid_constant__ Fp8Layout l, bool vec) {
  extern __shared__ __align__(16) float4 smem[];
  const int M = (int)p.M, pieces = (int)(l.kp >> 4), blocks = (int)l.blocks;
  uint32_t *scales = reinterpret_cast<uint32_t *>(smem + (size_t)M * pieces * 4);
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  int64_t n = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);

  Step w[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (n < p.N) w[i].load(p, n, i * kStepValues + lane * 16, l);
  stage_rows<T, kCodes>(p, x, ld, M, l, vec, smem, scales);
  __syncthreads();
  for (; n < p.N; n += warps) {
    float acc[kM];
#pragma unroll
    for (int m = 0; m < kM; ++m) acc[m] = 0.0f;
    for (int64_t k0 = 0; k0 < l.kp; k0 += kAhead * kStepValues) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t k = k0 + i * kStepValues + lane * 16;
        const Step s = w[i];
        // this slot's next piece: further along the row, or of the next row
        if (k0 + kAhead * kStepValues < l.kp)
          w[i].load(p, n, k + kAhead * kStepValues, l);
        else if (n + warps < p.N)
          w[i].load(p, n + warps, i * kStepValues + lane * 16, l);
        if (k >= l.kp) continue;
        float c[16];
        e4m3_values(s.codes.x, c);
        e4m3_values(s.codes.y, c + 4);
        e4m3_values(s.codes.z, c + 8);
        e4m3_values(s.codes.w, c + 12);
#pragma unroll
        for (int m = 0; m < kM; ++m) {
          if (m >= M) break;
          const float4 *v = smem + m * pieces * 4 + (k >> 4);
          float t = 0.0f, u = 0.0f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 f = v[q * pieces];
            t = __fmaf_rn(c[4 * q], f.x, t);
            u = __fmaf_rn(c[4 * q + 1], f.y, u);
            t = __fmaf_rn(c[4 * q + 2], f.z, t);
            u = __fmaf_rn(c[4 * q + 3], f.w, u);
          }
          acc[m] = add_scaled(acc[m], t + u, s.scale, scales[m * blocks + k / kFp8Block]);
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
        if (p.bias) v += load_as_f32(p.bias, p.bias_dtype, n);
        store_as(p.out, p.out_dtype, m * p.N + n, v);
      }
    }
  }
}

template <typename T, bool kCodes, int kM>
cudaError_t launch(const Fp8Product &p, const void *x, int64_t ld, const Fp8Layout &l,
                   cudaStream_t s) {
  auto kern = fp8_thin_kernel<T, kCodes, kM>;
  const size_t smem = (size_t)p.M * (l.kp * 4 + l.blocks * 4);
  if (smem > 48 * 1024) {
    // (always the most that this kernel uses: calls at the same time agree on it)
    const cudaError_t e = cudaFuncSetAttribute(
        kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
        kM * (SCMP_FP8_THIN_K * 4 + SCMP_FP8_THIN_K / kFp8Block * 4));
    if (e != cudaSuccess) return e;
  }
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld * (int)sizeof(T) % 16 == 0;
  const int64_t blocks = (p.N + kThreads / 32 - 1) / (kThreads / 32);
  // blocks that are resident together, less a prologue for each that waits: four per SM
  // for one row, two for more ([6144, 6144] 1: 15.8 us, with two 19.4; [4096, 4096] 2: 13.0,
  // with four 15.7; [4096, 1024] 4: 7.1, 8.8)
  const int64_t most = 148 * (kM == 1 ? 4 : 2);
  kern<<<(unsigned)(blocks < most ? blocks : most), kThreads, smem, s>>>(
      p, static_cast<const T *>(x), ld, l, vec);
  return cudaGetLastError();
}
template <typename T, bool kCodes>
cudaError_t launch_m(const Fp8Product &p, const void *x, int64_t ld, const Fp8Layout &l,
                     cudaStream_t s) {
  if (p.M == 1) return launch<T, kCodes, 1>(p, x, ld, l, s);
  return launch<T, kCodes, SCMP_FP8_THIN_ROWS>(p, x, ld, l, s);
}

}  // namespace

bool fp8_thin_fits(int64_t M, int64_t K) { return M <= SCMP_FP8_THIN_ROWS && K <= SCMP_FP8_THIN_K; }

// With k = K / 1024 and n = N / 1024 this launch takes about 2 + k n (0.13 + 0.17 M)
// + k (0.2 + 0.2 M) us, quantise + tensor-core tiles 5.2 + 1.8 k + 0.1 k n.  [N, K]
// and rows, this / the other (us, weights from HBM):
//   [1024, 1024]  1: 2.6 / 6.9   4: 4.1 / 6.9     [4096, 1024]  1: 4.2 / 8.3   4: 7.1 / 8.3
//   [1024, 4096]  1: 6.2 / 13.0  4: 10.6 / 13.0   [4096, 4096]  1: 9.3 / 13.5  2: 13.0 / 13.5
//   [16384, 1024] 1: 8.0 / 9.5   2: 11.5 / 9.5    [6144, 6144]  1: 15.9 / 17.9 2: 24.4 / 17.9
bool fp8_thin(int64_t M, int64_t N, int64_t K) {
  return fp8_thin_fits(M, K) &&
         K / 1024.0 * (N / 1024.0 * (0.03 + 0.17 * M) + 0.2 * M - 1.6) < 3.2;
}

cudaError_t launch_fp8_thin(const Fp8Product &p, const void *x, int x_dtype, int64_t ld,
                            cudaStream_t s) {
  const Fp8Layout l = fp8_layout(p.M, p.K);
  if (!x) return launch_m<float, true>(p, nullptr, 0, l, s);
  if (x_dtype == SCMP_F32) return launch_m<float, false>(p, x, ld, l, s);
  if (x_dtype == SCMP_BF16) return launch_m<__nv_bfloat16, false>(p, x, ld, l, s);
  return launch_m<__half, false>(p, x, ld, l, s);
}

}  // namespace scmp
