// Quantisation to 8-bit floating point with a scale per block of 128, and back.
//
// Rows alone: a warp takes 512 or 1024 columns of a row, a half-warp a block.
// With the transpose, or in squares: a block of threads takes a 128 x 128 tile,
// which it reads once; its columns' codes leave through shared memory as rows of
// the transpose.  Rows are bound by HBM, read once and written once (bf16 16448 x 4096:
// 37 us, 5.5 TB/s; fp32 51 us, 6.6 TB/s; back to bf16 33 us); tiles by instructions, two
// roundings and the search for two scales per element (bf16 both orders 45 us where the
// bytes take 41, squares in both 45, squares alone 32; fp32, two blocks an SM, 67 and 64
// where they take 62, squares alone 51).
#include "chunk.cuh"
#include "f32x2.cuh"
#include "fp8_common.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;

// ------------------------------------------------------------ rows alone

// A unit is kChunks x 256 columns of one row, one warp; a block's largest magnitude
// is a maximum over 16 lanes, and a lane writes the scales of four blocks at once.
template <typename T, bool kVec, int kChunks>
__global__ void __launch_bounds__(kThreads)
    fp8_rows_kernel(const T *__restrict__ x, int64_t ld, const __grid_constant__ Fp8Layout l,
                    const __grid_constant__ FastDiv per_row, uint32_t units,
                    uint8_t *__restrict__ data, uint8_t *__restrict__ scales) {
  __shared__ __align__(16) T deal[kVec ? 8 : kThreads * 8];
  // (a product behind this launch may set up as SMs become free)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  T *const buf = deal + (kVec ? 0 : (threadIdx.x >> 5) * 256);
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint64_t u = (blockIdx.x * kThreads + threadIdx.x) >> 5; u < units; u += warps) {
    const uint32_t r = per_row.quotient((uint32_t)u);
    const uint32_t chunk0 = ((uint32_t)u - r * per_row.d) * kChunks;
    const int64_t k = (int64_t)chunk0 * 256 + lane * 8;
    const bool live = r < l.rows;
    const T *row = x + r * ld;
    uint8_t *codes_at = data + r * l.kp + k;
    Chunk<T, kVec> e[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) e[i].load(row, (int64_t)(chunk0 + i) * 256, lane, l.K, live);
    uint32_t word[kChunks / 2];  // this half-warp's two bytes of each scale word
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      e[i].deal(buf, lane);
      float v[8];
      unpack16<T>(e[i].u[0], v);
      if (sizeof(T) == 4) unpack16<T>(e[i].u[sizeof(T) / 4], v + 4);
      uint32_t amax = max_bits8<T>(e[i].u[0], v);
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) amax = max(amax, __shfl_xor_sync(~0u, amax, o));
      const uint32_t b = 2 * (chunk0 + i) + (lane >> 4);
      const uint32_t scale = live && b < l.blocks ? fp8_scale(amax) : 0u;
      const float inv = fp8_inverse(scale);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= inv;
      const uint2 codes =
          make_uint2(e4m3x4(v[0], v[1], v[2], v[3]), e4m3x4(v[4], v[5], v[6], v[7]));
      if (live && k + i * 256 < l.kp) *reinterpret_cast<uint2 *>(codes_at + i * 256) = codes;
      const uint32_t both = scale | __shfl_xor_sync(~0u, scale, 16) << 8;  // (right in lane 0)
      if (i % 2 == 0)
        word[i / 2] = both;
      else
        word[i / 2] |= both << 16;
    }
#pragma unroll
    for (int i = 0; i < kChunks / 2; ++i) {
      const int64_t g = chunk0 / 2 + i;
      if (lane == 0 && g < l.groups)
        *reinterpret_cast<uint32_t *>(scales + mx_scale_word(r, g, l.groups)) = word[i];
    }
  }
}

// -------------------------------------------- tiles: both orders, or squares

struct TileArgs {
  Fp8Layout rows, cols;  // of x and of its transpose
  int64_t ld;
  uint8_t *data, *scales, *t_data, *t_scales;  // either pair nullable
  float *column_sums;                          // nullable
  FastDiv tiles_c{1};
};

// Largest magnitudes: 32-bit patterns of fp32, whose order is the numbers' with every
// NaN above the infinities; pairs of 16-bit numbers as such, where a NaN wins too.
template <typename T> struct Magnitude {
  static constexpr int kWords = 8 * (int)sizeof(T) / 4;  // of eight elements
  // of m (magnitudes) and the values of w
  static __device__ __forceinline__ uint32_t most(uint32_t m, uint32_t w) {
    if constexpr (sizeof(T) == 4) {
      return max(m, w & 0x7FFFFFFFu);
    } else if constexpr (__is_same(T, __nv_bfloat16)) {
      const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162 *>(&m),
                                           __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&w)));
      return *reinterpret_cast<const uint32_t *>(&r);
    } else {
      const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2 *>(&m),
                                    __habs2(*reinterpret_cast<const __half2 *>(&w)));
      return *reinterpret_cast<const uint32_t *>(&r);
    }
  }
  // bits of the fp32 magnitude in the low half (or the word)
  static __device__ __forceinline__ uint32_t bits(uint32_t m) {
    if (sizeof(T) == 4) return m;
    if (__is_same(T, __nv_bfloat16)) return m << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
  }
};

// Thread t holds rows 8 (t / 16) + i and columns 8 (t % 16) + j of the tile, i, j < 8.
// The transpose is kept in shared memory as 128 rows of 16 pieces of 8 bytes, piece u
// of row c at u ^ (c / 8 % 16): what 16 threads store at a time, 8 rows apart, and
// what they load along a row both spread over all banks (in plain order the stores'
// conflicts took the bf16 tile of 128 x 128 from 4 to 12 us).
// (16-bit tiles in both orders with three blocks an SM 53 us, with four 50, and 45 since
// each scale is found by one thread instead of sixteen; with sums or unaligned, four would
// spill: a step with a bias 2 us more)
template <typename T, bool kVec, bool kSquare, bool kSums>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : kVec && !kSums ? 4 : 3)
    fp8_tile_kernel(const T *__restrict__ x, const __grid_constant__ TileArgs a) {
  using Mag = Magnitude<T>;
  constexpr int kWords = Mag::kWords;
  __shared__ __align__(16) uint8_t turned[128 * 128];
  __shared__ __align__(16) uint32_t warp_max[8][16 * kWords];
  __shared__ __align__(16) float warp_sum[kSums ? 8 : 1][128];
  __shared__ __align__(16) float col_inv[128];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rg = threadIdx.x >> 4, piece = threadIdx.x & 15;
  const uint32_t tile_row = a.tiles_c.quotient(blockIdx.x);
  const int64_t tile_r = tile_row, tile_c = blockIdx.x - tile_row * a.tiles_c.d;
  const int64_t r0 = tile_r * 128 + rg * 8, c0 = tile_c * 128 + piece * 8;
  const int64_t rows = a.rows.rows, K = a.rows.K;

  // the tile, as loaded
  uint32_t e[8][kWords];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const T *p = x + (r0 + i) * a.ld + c0;
    if (kVec && r0 + i < rows && c0 + 8 <= K) {
#pragma unroll
      for (int h = 0; h < kWords / 4; ++h) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p) + h);
        e[i][4 * h] = u.x;
        e[i][4 * h + 1] = u.y;
        e[i][4 * h + 2] = u.z;
        e[i][4 * h + 3] = u.w;
      }
    } else {
      T v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = r0 + i < rows && c0 + j < K ? p[j] : from_f32<T>(0.0f);
      memcpy(e[i], v, sizeof(v));
    }
  }
  // columns j and j + 1 (j even) of row i
  const auto two = [&](int i, int j) {
    if constexpr (sizeof(T) == 4)
      return make_float2(__uint_as_float(e[i][j]), __uint_as_float(e[i][j + 1]));
    else
      return unpack2<T>(e[i][j / 2]);
  };

  // largest magnitudes: of the thread's part of each row and of each column
  uint32_t row_max[8], col_max[kWords];
#pragma unroll
  for (int w = 0; w < kWords; ++w) col_max[w] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      m = Mag::most(m, e[i][w]);
      col_max[w] = Mag::most(col_max[w], e[i][w]);
    }
    row_max[i] = sizeof(T) == 4 ? m : Mag::most(m, __funnelshift_r(m, m, 16));
  }
  // scales: of a row from the lane of its number (the half-warp's rows), of a column from
  // the thread of its number, others get what to multiply by
  uint32_t row_scale = 0, square_scale = 0;
  float row_inv[8];
  if (kSquare) {
    uint32_t m = row_max[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = Mag::most(m, row_max[i]);
    m = __reduce_max_sync(~0u, sizeof(T) == 4 ? m : m & 0xFFFFu);  // (a NaN's pattern is the largest)
    if (lane == 0) warp_max[0][warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, warp_max[0][w]);
    row_scale = square_scale = fp8_scale(Mag::bits(m));
#pragma unroll
    for (int i = 0; i < 8; ++i) row_inv[i] = fp8_inverse(row_scale);
  } else {
    if (a.data) {
      uint32_t m = 0;  // of row piece % 8
      if constexpr (sizeof(T) == 2) {  // two rows at a time
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          uint32_t u = __byte_perm(row_max[i], row_max[i + 1], 0x5410);
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) u = Mag::most(u, __shfl_xor_sync(~0u, u, o));
          if ((piece & 6) == i) m = u;
        }
        m = piece & 1 ? m >> 16 : m & 0xFFFFu;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t u = row_max[i];
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) u = max(u, __shfl_xor_sync(~0u, u, o));
          if ((piece & 7) == i) m = u;
        }
      }
      row_scale = fp8_scale(Mag::bits(m));
      const float inv = fp8_inverse(row_scale);
#pragma unroll
      for (int i = 0; i < 8; ++i) row_inv[i] = __shfl_sync(~0u, inv, (lane & 16) + i);
    }
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      col_max[w] = Mag::most(col_max[w], __shfl_xor_sync(~0u, col_max[w], 16));
    if (lane < 16) {
#pragma unroll
      for (int w = 0; w < kWords; w += 4)
        *reinterpret_cast<uint4 *>(&warp_max[warp][piece * kWords + w]) =
            make_uint4(col_max[w], col_max[w + 1], col_max[w + 2], col_max[w + 3]);
    }
    if (kSums) {
      float2 sums[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sums[j] = two(0, 2 * j);
#pragma unroll
        for (int i = 1; i < 8; ++i) {
          const float2 v = two(i, 2 * j);
          sums[j].x += v.x;
          sums[j].y += v.y;
        }
        sums[j].x += __shfl_xor_sync(~0u, sums[j].x, 16);
        sums[j].y += __shfl_xor_sync(~0u, sums[j].y, 16);
      }
      if (lane < 16) {
        float4 *to = reinterpret_cast<float4 *>(&warp_sum[warp][piece * 8]);
        to[0] = make_float4(sums[0].x, sums[0].y, sums[1].x, sums[1].y);
        to[1] = make_float4(sums[2].x, sums[2].y, sums[3].x, sums[3].y);
      }
    }
    __syncthreads();
    if (a.t_data && threadIdx.x < 128) {
      uint32_t m = 0;  // (patterns of magnitudes, a NaN's the largest)
#pragma unroll
      for (int q = 0; q < 8; ++q)
        m = max(m, sizeof(T) == 4
                       ? warp_max[q][threadIdx.x]
                       : (uint32_t) reinterpret_cast<const uint16_t *>(warp_max[q])[threadIdx.x]);
      const uint32_t scale = fp8_scale(Mag::bits(m));
      const int64_t c = tile_c * 128 + threadIdx.x;
      col_inv[threadIdx.x] = fp8_inverse(scale);
      a.t_scales[fp8_scale_at(c, tile_r, a.cols.groups)] = (uint8_t)(c < K ? scale : 0u);
    }
    if (kSums && threadIdx.x < 128 && tile_c * 128 + threadIdx.x < K) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += warp_sum[w][threadIdx.x];
      a.column_sums[tile_r * K + tile_c * 128 + threadIdx.x] = t;
    }
  }

  const int live_r = (int)(rows - r0 < 8 ? rows - r0 : 8);
  if (a.data) {
    uint8_t *to = a.data + r0 * a.rows.kp + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i, to += a.rows.kp) {
      uint32_t codes[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 u = mul2(two(i, 4 * h), both(row_inv[i])),
                     w = mul2(two(i, 4 * h + 2), both(row_inv[i]));
        codes[h] = e4m3x4(u.x, u.y, w.x, w.y);
      }
      if (i < live_r)  // (columns up to the end of the block are the row's)
        *reinterpret_cast<uint2 *>(to) = make_uint2(codes[0], codes[1]);
    }
    if (piece < 8)  // (eight rows of a scale atom are 16 bytes apart)
      a.scales[fp8_scale_at(r0, tile_c, a.rows.groups) + 16 * piece] =
          (uint8_t)(piece < live_r ? row_scale : 0u);
    // the last tile of a row also fills its last scale word
    if (tile_c == a.rows.blocks - 1 && threadIdx.x < 128)
      for (int64_t b = a.rows.blocks; b < a.rows.groups * 4; ++b)
        a.scales[fp8_scale_at(tile_r * 128 + threadIdx.x, b, a.rows.groups)] = 0;
  }
  if (a.t_data) {
    if (!kSquare) __syncthreads();  // col_inv
    // column j's eight rows are eight neighbouring bytes of the transpose
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 inv = kSquare ? both(row_inv[0])
                                 : *reinterpret_cast<const float2 *>(&col_inv[piece * 8 + j]);
      uint32_t u[2], w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 p = mul2(two(4 * h, j), inv), q = mul2(two(4 * h + 1, j), inv),
                     r = mul2(two(4 * h + 2, j), inv), t = mul2(two(4 * h + 3, j), inv);
        u[h] = e4m3x4(p.x, q.x, r.x, t.x);
        w[h] = e4m3x4(p.y, q.y, r.y, t.y);
      }
      uint8_t *at = turned + (piece * 8 + j) * 128 + (rg ^ piece) * 8;
      *reinterpret_cast<uint2 *>(at) = make_uint2(u[0], u[1]);
      *reinterpret_cast<uint2 *>(at + 128) = make_uint2(w[0], w[1]);
    }
    if (kSquare && threadIdx.x < 128) {
      const int64_t c = tile_c * 128 + threadIdx.x;
      a.t_scales[fp8_scale_at(c, tile_r, a.cols.groups)] = (uint8_t)(c < K ? square_scale : 0u);
    }
    if (tile_r == a.cols.blocks - 1 && threadIdx.x < 128)
      for (int64_t b = a.cols.blocks; b < a.cols.groups * 4; ++b)
        a.t_scales[fp8_scale_at(tile_c * 128 + threadIdx.x, b, a.cols.groups)] = 0;
    __syncthreads();
    const int m = threadIdx.x & 7, left = (int)(K - tile_c * 128 < 128 ? K - tile_c * 128 : 128);
    uint8_t *to = a.t_data + (tile_c * 128 + (threadIdx.x >> 3)) * a.cols.kp + tile_r * 128 + m * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i, to += 32 * a.cols.kp) {
      const int c = (threadIdx.x >> 3) + i * 32, at = c >> 3;
      uint4 v = *reinterpret_cast<const uint4 *>(turned + c * 128 + (m ^ at >> 1) * 16);
      if (at & 1) v = make_uint4(v.z, v.w, v.x, v.y);
      if (c < left) *reinterpret_cast<uint4 *>(to) = v;
    }
  }
}

// Sums of columns over the tiles' parts, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(512)
    fp8_sum_kernel(const float *__restrict__ sums, int64_t parts, int64_t K, T *__restrict__ out) {
  // 32 columns, a thread of each of 16 warps: part p of a column goes to warp p % 16
  __shared__ float part[16][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float t = 0.0f;
  if (c < K) {
#pragma unroll 8
    for (int64_t p = w; p < parts; p += 16) t += sums[p * K + c];
  }
  part[w][lane] = t;
  __syncthreads();
  if (w == 0 && c < K) {
    t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += part[i][lane];
    out[c] = from_f32<T>(t);
  }
}

// ------------------------------------------------------------------- back

// Eight (16-bit) or four (fp32) consecutive elements per lane and chunk of 32 lanes.
template <typename T, int kChunks, bool kVec>
__global__ void __launch_bounds__(kThreads)
    fp8_values_kernel(const uint8_t *__restrict__ data, const uint8_t *__restrict__ scales,
                      const __grid_constant__ Fp8Layout l, const __grid_constant__ FastDiv per_row,
                      uint32_t units, T *__restrict__ out) {
  constexpr int V = kVec16<T>;
  __shared__ __align__(16) T deal[kVec ? 8 : kThreads * V];
  const int lane = threadIdx.x & 31;
  T *const buf = deal + (kVec ? 0 : (threadIdx.x >> 5) * 32 * V);
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint64_t u = (blockIdx.x * kThreads + threadIdx.x) >> 5; u < units; u += warps) {
    const uint32_t r = per_row.quotient((uint32_t)u);
    const int64_t k = ((int64_t)((uint32_t)u - r * per_row.d) * kChunks * 32 + lane) * V;
    uint32_t codes[kChunks][V / 4], sc[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int64_t ki = k + i * 32 * V;
      sc[i] = 0;
#pragma unroll
      for (int j = 0; j < V / 4; ++j) codes[i][j] = 0;
      if (ki < l.kp) {
#pragma unroll
        for (int j = 0; j < V / 4; ++j)
          codes[i][j] = __ldg(reinterpret_cast<const uint32_t *>(data + r * l.kp + ki) + j);
        sc[i] = __ldg(scales + fp8_scale_at(r, ki / kFp8Block, l.groups));
      }
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int64_t ki = k + i * 32 * V;
      if (ki - lane * V >= l.K) break;
      const float s = fp8_value_of_scale(sc[i]);
      float v[V];
#pragma unroll
      for (int j = 0; j < V / 4; ++j) e4m3_values(codes[i][j], v + 4 * j);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= s;
      T *dst = out + r * l.K + ki;
      if (kVec) {
        if (ki < l.K) *reinterpret_cast<uint4 *>(dst) = pack16<T>(v);
      } else {
        *reinterpret_cast<uint4 *>(buf + lane * V) = pack16<T>(v);
        __syncwarp();
        const int64_t c = ki - lane * V + lane;  // a neighbour per lane
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + 32 * j < l.K) out[r * l.K + c + 32 * j] = buf[lane + 32 * j];
        __syncwarp();
      }
    }
  }
}

unsigned grid_for(uint32_t units) {
  const int64_t b = ((int64_t)units + kThreads / 32 - 1) / (kThreads / 32);
  return (unsigned)(b < 148 * 16 ? b : 148 * 16);
}

// (rows and their units stay below 2^32 for what fits the memory)
template <typename T, bool kVec, int kChunks>
cudaError_t rows_k(const Fp8Quantize &q, const Fp8Layout &l, cudaStream_t s) {
  const FastDiv per_row((uint32_t)((l.kp + 256 * kChunks - 1) / (256 * kChunks)));
  const uint32_t units = (uint32_t)((l.rows + 127) / 128 * 128) * per_row.d;
  fp8_rows_kernel<T, kVec, kChunks><<<grid_for(units), kThreads, 0, s>>>(
      static_cast<const T *>(q.x), q.ld, l, per_row, units, q.data, q.scales);
  return cudaGetLastError();
}
template <typename T, bool kVec>
cudaError_t tiles_k(const Fp8Quantize &q, cudaStream_t s) {
  TileArgs a;
  a.rows = fp8_layout(q.rows, q.K);
  a.cols = fp8_layout(q.K, q.rows);
  a.ld = q.ld;
  a.data = q.data;
  a.scales = q.scales;
  a.t_data = q.t_data;
  a.t_scales = q.t_scales;
  a.column_sums = q.column_sums;
  a.tiles_c = FastDiv((uint32_t)a.rows.blocks);
  const int64_t tiles = a.rows.blocks * a.cols.blocks;
  if (tiles > INT32_MAX) return cudaErrorInvalidConfiguration;
  const unsigned grid = (unsigned)tiles;
  const T *x = static_cast<const T *>(q.x);
  if (q.square)
    fp8_tile_kernel<T, kVec, true, false><<<grid, kThreads, 0, s>>>(x, a);
  else if (q.column_sums)
    fp8_tile_kernel<T, kVec, false, true><<<grid, kThreads, 0, s>>>(x, a);
  else
    fp8_tile_kernel<T, kVec, false, false><<<grid, kThreads, 0, s>>>(x, a);
  return cudaGetLastError();
}
template <typename T> cudaError_t quantize(const Fp8Quantize &q, cudaStream_t s) {
  const bool vec =
      (reinterpret_cast<uintptr_t>(q.x) & 15) == 0 && (q.ld * (int64_t)sizeof(T)) % 16 == 0;
  if (q.square || q.t_data || q.column_sums)
    return vec ? tiles_k<T, true>(q, s) : tiles_k<T, false>(q, s);
  const Fp8Layout l = fp8_layout(q.rows, q.K);
  // Four chunks in flight per warp for 16-bit types, unless that pads rows further
  // than two do (bf16, four / two: 16448 x 4096 37 / 42 us, 16448 x 1024 11.0 / 11.6,
  // 40000 x 384 28.8 / 16.1, 2000 x 1030 5.7 / 4.6); two are enough for fp32 (51 / 51, 14.1 /
  // 13.1).
  if constexpr (sizeof(T) == 2)
    if ((l.kp + 1023) / 1024 * 2 == (l.kp + 511) / 512)
      return vec ? rows_k<T, true, 4>(q, l, s) : rows_k<T, false, 4>(q, l, s);
  return vec ? rows_k<T, true, 2>(q, l, s) : rows_k<T, false, 2>(q, l, s);
}

template <typename T, int kChunks, bool kVec>
cudaError_t values_v(const uint8_t *data, const uint8_t *scales, const Fp8Layout &l, void *out,
                     cudaStream_t s) {
  constexpr int V = kVec16<T>;
  const FastDiv per_row((uint32_t)((l.kp + 32 * V * kChunks - 1) / (32 * V * kChunks)));
  const uint32_t units = (uint32_t)l.rows * per_row.d;
  fp8_values_kernel<T, kChunks, kVec><<<grid_for(units), kThreads, 0, s>>>(
      data, scales, l, per_row, units, static_cast<T *>(out));
  return cudaGetLastError();
}
template <typename T>
cudaError_t values_t(const uint8_t *data, const uint8_t *scales, const Fp8Layout &l, void *out,
                     cudaStream_t s) {
  const bool vec = l.K % kVec16<T> == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  return vec ? values_v<T, 4, true>(data, scales, l, out, s)
             : values_v<T, 4, false>(data, scales, l, out, s);
}

}  // namespace

cudaError_t launch_fp8_quantize(const Fp8Quantize &q, cudaStream_t s) {
  if (q.dtype == SCMP_F32) return quantize<float>(q, s);
  if (q.dtype == SCMP_BF16) return quantize<__nv_bfloat16>(q, s);
  return quantize<__half>(q, s);
}

cudaError_t launch_fp8_dequantize(const uint8_t *data, const uint8_t *scales, const Fp8Layout &l,
                                  void *out, int dtype, cudaStream_t s) {
  if (dtype == SCMP_F32) return values_t<float>(data, scales, l, out, s);
  if (dtype == SCMP_BF16) return values_t<__nv_bfloat16>(data, scales, l, out, s);
  return values_t<__half>(data, scales, l, out, s);
}

cudaError_t launch_fp8_sum_columns(const float *sums, int64_t parts, int64_t K, void *out,
                                   int dtype, cudaStream_t s) {
  const unsigned grid = (unsigned)((K + 31) / 32);
  if (dtype == SCMP_F32)
    fp8_sum_kernel<float><<<grid, 512, 0, s>>>(sums, parts, K, static_cast<float *>(out));
  else if (dtype == SCMP_BF16)
    fp8_sum_kernel<__nv_bfloat16>
        <<<grid, 512, 0, s>>>(sums, parts, K, static_cast<__nv_bfloat16 *>(out));
  else
    fp8_sum_kernel<__half><<<grid, 512, 0, s>>>(sums, parts, K, static_cast<__half *>(out));
  return cudaGetLastError();
}

}  // namespace scmp
