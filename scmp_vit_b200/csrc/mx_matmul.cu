// Product of two microscaled 4-bit operands on the tensor cores:
//   out[m, n] = 2^e sum_k A[m, k] B[n, k] (+ bias[n]),
// A [M, K] activations, B [N, K] a weight, both in the layout of mx_common.cuh.
//
// tcgen05.mma kind::mxf4 / kind::mxf4nvf4 on CTA pairs (cta_group::2): 256
// weight rows are the accumulator's lanes (128 per CTA), `nt` activation rows
// its columns, so that a lane owns one output feature (its bias is one
// register) and 32 lanes store 32 neighbouring outputs.  Each 256-value step of
// K is one stage of a shared-memory ring that a TMA thread per CTA fills: both
// operands' codes (128-byte rows, 128-byte swizzle) and their scale atoms,
// which tcgen05.cp moves into tensor memory in front of the step's MMAs.  Two
// accumulators of up to 192 columns alternate, so the epilogue of one tile runs
// under the MMAs of the next; the scales use the columns behind them.
//
// Warps: 0 loads, 1 issues MMAs (even CTA) or forwards "stage full" to the even
// CTA (odd CTA), 2 owns the tensor memory, 4-7 run the epilogue.  Every wait is
// bounded: a wait that gives up raises the error word and the pair drains.
#include "mx_common.cuh"
#include "tc_ptx.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 256;
constexpr int kStages = 6;
constexpr int kMaxNt = 192;        // activation rows per tile
constexpr uint32_t kStepBytes = 128;  // bytes of a row per stage: 256 values
constexpr uint32_t kAccCols = kMaxNt;
constexpr uint32_t kScaleCol = 2 * kAccCols;

template <int kFmt> struct MxCfg {
  static constexpr int kGroups = kFmt == SCMP_MXFP4 ? 2 : 4;  // scale atoms per stage and row group
  static constexpr uint32_t kW = 128 * kStepBytes;            // a CTA's weight rows
  static constexpr uint32_t kX = kMaxNt / 2 * kStepBytes;     // a CTA's activation rows
  static constexpr uint32_t kWs = kGroups * 512;
  static constexpr uint32_t kXs = 2 * kGroups * 512;  // a tile's rows touch two row groups at most
  static constexpr uint32_t kStage = kW + kX + kWs + kXs;
  static constexpr uint32_t kScaleCols = kGroups * 4 + kGroups * 8;
  static constexpr size_t kSmem = (size_t)kStages * kStage + 1024 /*align*/ + 256;
  static_assert(kStage % 1024 == 0, "swizzle atoms stay aligned");
  static_assert(kScaleCol + 2 * kScaleCols <= 512, "two sets of scales behind the accumulators");
  static_assert(kSmem <= 227 * 1024, "shared memory per CTA");
};

struct MxTiles {
  MxProduct p;
  int nt;                  // activation rows per tile (16, 32, 64, 128 or 192)
  int64_t tiles_f, tiles;  // weight tiles (256 rows); all tiles, weight tiles fastest
  int64_t groups;          // scale atoms along K
  int steps;               // stages per tile
  int mmas;                // 64-value MMAs per tile
  unsigned int *error;
};

template <int kFmt> __host__ __device__ constexpr uint32_t idesc(int n, int sf_id) {
  return (1u << 7)                                     // A e2m1
         | (1u << 10)                                  // B e2m1
         | ((uint32_t)(n >> 3) << 17)                  // N
         | ((kFmt == SCMP_MXFP4 ? 1u : 0u) << 23)      // scales e8m0 / e4m3
         | ((uint32_t)(256 >> 4) << 24)                // M over the pair
         | ((uint32_t)sf_id << 4) | ((uint32_t)sf_id << 29);  // byte of the scale word
}
template <int kFmt>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if (kFmt == SCMP_MXFP4)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], "
        "p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], "
        "[%6], p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
}
// One scale atom: 32 lanes x 16 bytes of shared memory to four columns of every
// lane quarter, in both CTAs from the same offset.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}
// Unswizzled descriptor of 8-row x 16-byte pieces 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(128u >> 4) << 32 | (uint64_t)1 << 46;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes,
                                          uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ float load_as_f32(const void *p, int dtype, int64_t i) {
  if (dtype == SCMP_F32) return static_cast<const float *>(p)[i];
  if (dtype == SCMP_BF16) return to_f32(static_cast<const __nv_bfloat16 *>(p)[i]);
  return to_f32(static_cast<const __half *>(p)[i]);
}

struct Coord {
  int64_t f0, n0;  // first weight row (of this CTA), first activation row
  int xg, nxg;     // first row group of the activations' scales, how many exist
};
__device__ __forceinline__ Coord coord(const MxTiles &t, int64_t tile, uint32_t rank) {
  Coord c;
  c.f0 = tile % t.tiles_f * 256 + rank * 128;
  c.n0 = tile / t.tiles_f * t.nt;
  c.xg = (int)(c.n0 >> 7);
  const int touched = ((int)(c.n0 & 127) + t.nt + 127) >> 7;
  const int64_t left = ((t.p.M + 127) >> 7) - c.xg;
  c.nxg = left < touched ? (int)left : touched;
  return c;
}

template <int kFmt, typename T>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    mx_pair_kernel(const __grid_constant__ MxTiles t, const __grid_constant__ CUtensorMap wmap,
                   const __grid_constant__ CUtensorMap xmap) {
  using Cfg = MxCfg<kFmt>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kStages * Cfg::kStage);
  uint64_t *empty = full + kStages, *pfull = empty + kStages;
  uint64_t *tfull = pfull + kStages, *tempty = tfull + 2, *drain = tempty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);   // this CTA's loader
      mbar_init(&empty[s], 1);  // commit of the MMAs that read the stage
      mbar_init(&pfull[s], 1);  // even CTA: the odd CTA's stage is full
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 8);  // even CTA: the epilogue warps of both
    }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers and tensor memory exist
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  const uint32_t smem0 = smem_u32(smem);

  if (warp == 0 && lane == 0) {
    // -------------------------------------------------------------- loader
    int stage = 0;
    uint32_t phase = 0;
    int64_t issued = 0;
    const uint32_t x_bytes = (uint32_t)t.nt / 2 * kStepBytes;
    const int64_t w_groups = (t.p.N + 127) >> 7;
    bool ok = producers_released(abort);
    for (int64_t tile = cluster; tile < t.tiles && ok; tile += clusters) {
      const Coord c = coord(t, tile, rank);
      const bool has_w = (c.f0 >> 7) < w_groups;
      const uint8_t *ws = t.p.b_scales + (c.f0 >> 7) * t.groups * 512;
      const uint8_t *xs = t.p.a_scales + c.xg * t.groups * 512;
      for (int kb = 0; kb < t.steps; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort)) {
          ok = false;
          break;
        }
        const int64_t g0 = (int64_t)kb * Cfg::kGroups;
        const int64_t left = t.groups - g0;
        const uint32_t sf = (uint32_t)(left < Cfg::kGroups ? left : Cfg::kGroups) * 512;
        const uint32_t at = smem0 + stage * Cfg::kStage;
        // rows past an operand's end arrive as zeros and count as bytes
        mbar_arrive_expect_tx(&full[stage],
                              Cfg::kW + x_bytes + sf * (uint32_t)(c.nxg + (has_w ? 1 : 0)));
        tma_load_2d(at, &wmap, kb * (int)kStepBytes, (int)c.f0, &full[stage]);
        tma_load_2d(at + Cfg::kW, &xmap, kb * (int)kStepBytes,
                    (int)(c.n0 + rank * (uint32_t)(t.nt / 2)), &full[stage]);
        if (has_w) bulk_load(at + Cfg::kW + Cfg::kX, ws + g0 * 512, sf, &full[stage]);
        for (int r = 0; r < c.nxg; ++r)
          bulk_load(at + Cfg::kW + Cfg::kX + Cfg::kWs + r * (Cfg::kGroups * 512),
                    xs + (r * t.groups + g0) * 512, sf, &full[stage]);
        ++issued;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // no CTA ends with its own copies in flight
    for (int64_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
      mbar_wait_own(&full[i % kStages], (uint32_t)(i / kStages & 1));
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // --------------------------------------------------------- MMA issuer
    int stage = 0;
    uint32_t phase = 0, it = 0, set = 0;
    const uint64_t desc0 = smem_desc_sw128(smem0);
    const uint32_t id0 = idesc<kFmt>(t.nt, 0), id2 = idesc<kFmt>(t.nt, 2);
    bool ok = true;
    for (int64_t tile = cluster; tile < t.tiles && ok; tile += clusters, ++it) {
      const Coord c = coord(t, tile, 0);
      const uint32_t buf = it & 1;
      if (it >= 2 && !mbar_wait_cl(&tempty[buf], ((it >> 1) - 1) & 1, abort)) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * kAccCols;
      int left = t.mmas;
      for (int kb = 0; kb < t.steps; ++kb, left -= 4, set ^= 1) {
        if (!mbar_wait(&full[stage], phase, abort) || !mbar_wait_cl(&pfull[stage], phase, abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t base = smem0 + stage * Cfg::kStage;
        const uint32_t sw = tmem + kScaleCol + set * Cfg::kScaleCols, sx = sw + Cfg::kGroups * 4;
        const uint64_t dw = scale_desc(base + Cfg::kW + Cfg::kX);
#pragma unroll
        for (int g = 0; g < Cfg::kGroups; ++g) {
          if (g * (4 / Cfg::kGroups) >= left) break;  // past K
          copy_scales(sw + g * 4, desc_add(dw, g * 512));
          for (int r = 0; r < c.nxg; ++r)
            copy_scales(sx + g * 8 + r * 4,
                        desc_add(dw, Cfg::kWs + (r * Cfg::kGroups + g) * 512));
        }
        const uint64_t d = desc_add(desc0, (uint32_t)stage * Cfg::kStage);
        const uint32_t sxo = sx + ((uint32_t)c.n0 & 127u) / 32;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          if (kk >= left) break;
          const int g = kFmt == SCMP_MXFP4 ? kk >> 1 : kk;
          mma_pair<kFmt>(acc, desc_add(d, kk * 32), desc_add(d, Cfg::kW + kk * 32),
                         kFmt == SCMP_MXFP4 && (kk & 1) ? id2 : id0, sw + g * 4, sxo + g * 8,
                         (kb > 0 || kk > 0) ? 1u : 0u);
        }
        tc_commit_pair_both(&empty[stage]);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      tc_commit_pair_both(&tfull[buf]);
    }
    tc_commit_pair_local(drain);
    mbar_wait_own_cl(drain, 0);
  } else if (warp == 1 && lane == 0) {
    // -------------------------------- odd CTA: its stages' arrival, forwarded
    const uint32_t to = mapa_shared(smem_u32(pfull), 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int64_t tile = cluster; tile < t.tiles && ok; tile += clusters)
      for (int kb = 0; kb < t.steps; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort)) {
          ok = false;
          break;
        }
        mbar_arrive_cluster(to + 8u * (uint32_t)stage);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t to = mapa_shared(smem_u32(tempty), 0);
    T *const out = static_cast<T *>(t.p.out);
    uint32_t it = 0;
    for (int64_t tile = cluster; tile < t.tiles; tile += clusters, ++it) {
      const Coord c = coord(t, tile, rank);
      const uint32_t buf = it & 1;
      // one lane waits for all 32: they leave together when it gives up
      const bool ok = lane != 0 || mbar_wait(&tfull[buf], (it >> 1) & 1, abort);
      if (!__shfl_sync(~0u, (int)ok, 0)) break;
      tc_fence_after();
      const int64_t f = c.f0 + (warp & 3) * 32 + lane;
      const bool live = f < t.p.N;
      const float bias = t.p.bias && live ? load_as_f32(t.p.bias, t.p.bias_dtype, f) : 0.0f;
      const int64_t rows = t.p.M - c.n0;
      for (int j0 = 0; j0 < t.nt; j0 += 16) {
        uint32_t v[16];
        __syncwarp();
        tmem_ld16(tmem + lanes + buf * kAccCols + j0, v);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (j0 + 16 >= t.nt) {  // the accumulator is in registers: free for the next tile but one
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(to + 8u * buf);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (live && j0 + j < rows) {
            const float a = __uint_as_float(v[j]);
            out[(c.n0 + j0 + j) * t.p.N + f] =
                from_f32<T>(t.p.bias ? __fmaf_rn(a, t.p.alpha, bias) : a * t.p.alpha);
          }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while the pair may still touch its memory
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
  if (threadIdx.x == 0 && *abort) atomicOr(t.error, 1u);
}

bool encode_rows(CUtensorMap *map, const uint8_t *data, int64_t rows, int64_t row_bytes,
                 uint32_t box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  cuuint64_t gdim[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
  cuuint64_t gstride[1] = {(cuuint64_t)row_bytes};
  cuuint32_t box[2] = {kStepBytes, box_rows};
  cuuint32_t estride[2] = {1u, 1u};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(data), gdim, gstride,
             box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Activation rows per tile: one tile for up to 32 rows; else the width among
// 64, 128 and 192 whose rounds of tiles over the CTA pairs cost least, a tile
// costing its columns plus about 48 (its fixed part), the wider on a tie.
// (Starts of tiles are multiples of 64 rows: the scale columns they begin at
// are even.)
int tile_rows(int64_t M, int64_t tiles_f, int clusters) {
  if (M <= 16) return 16;
  if (M <= 32) return 32;
  int best = kMaxNt;
  int64_t best_cost = -1;
  for (int nt : {192, 128, 64}) {
    const int64_t tiles = tiles_f * ((M + nt - 1) / nt);
    const int64_t cost = (tiles + clusters - 1) / clusters * (nt + 48);
    if (best_cost < 0 || cost < best_cost) {
      best_cost = cost;
      best = nt;
    }
  }
  return best;
}

template <int kFmt, typename T>
cudaError_t launch(MxTiles t, int64_t kp, cudaStream_t s) {
  using Cfg = MxCfg<kFmt>;
  auto kern = mx_pair_kernel<kFmt, T>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)Cfg::kSmem)) != cudaSuccess)
    return e;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = s;
  // one cluster per resident pair slot (persistent tiles)
  static int max_clusters[kMaxCachedDevices] = {};
  int clusters = dev < kMaxCachedDevices ? max_clusters[dev] : 0;
  if (clusters <= 0) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(2, 1, 1);
    if ((e = cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg)) != cudaSuccess) return e;
    if (clusters <= 0) return cudaErrorInvalidConfiguration;
    if (dev < kMaxCachedDevices) max_clusters[dev] = clusters;
    cfg.attrs = nullptr;
    cfg.numAttrs = 0;
  }
  t.tiles_f = (t.p.N + 255) / 256;
  t.nt = tile_rows(t.p.M, t.tiles_f, clusters);
  t.tiles = t.tiles_f * ((t.p.M + t.nt - 1) / t.nt);
  t.steps = (int)((kp + 255) / 256);
  t.mmas = (int)((kp + 63) / 64);
  CUtensorMap wmap, xmap;
  if (!encode_rows(&wmap, t.p.b, t.p.N, kp / 2, 128) ||
      !encode_rows(&xmap, t.p.a, t.p.M, kp / 2, (uint32_t)t.nt / 2))
    return cudaErrorInvalidValue;
  const int64_t grid = t.tiles < clusters ? t.tiles : clusters;
  kern<<<(unsigned)(2 * grid), kThreads, Cfg::kSmem, s>>>(t, wmap, xmap);
  return cudaGetLastError();
}

template <int kFmt> cudaError_t launch_typed(const MxTiles &t, int64_t kp, cudaStream_t s) {
  if (t.p.out_dtype == SCMP_F32) return launch<kFmt, float>(t, kp, s);
  if (t.p.out_dtype == SCMP_BF16) return launch<kFmt, __nv_bfloat16>(t, kp, s);
  return launch<kFmt, __half>(t, kp, s);
}

}  // namespace

cudaError_t launch_mx_matmul(const MxProduct &p, unsigned int *error, cudaStream_t s,
                             int *launches) {
  *launches = 1;
  const MxLayout l = mx_layout(p.M, p.K, p.fmt);
  MxTiles t{};
  t.p = p;
  t.groups = l.groups;
  t.error = error;
  return p.fmt == SCMP_MXFP4 ? launch_typed<SCMP_MXFP4>(t, l.kp, s)
                             : launch_typed<SCMP_NVFP4>(t, l.kp, s);
}

cudaError_t mx_set_wait_limit(unsigned long long ns) {
  return cudaMemcpyToSymbol(g_wait_limit_ns, &ns, sizeof(ns));
}
cudaError_t mx_hold_producers(int on) {
  return cudaMemcpyToSymbol(g_hold_producers, &on, sizeof(on));
}

}  // namespace scmp
