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
// which tcgen05.cp moves into tensor memory in front of the step's MMAs.  Both
// CTAs' copies complete on the even CTA's barrier, which its MMA thread waits
// on (forwarding the odd CTA's arrivals by a thread held a stage to 0.58 us,
// three times its MMAs).  Two accumulators of up to 192 columns alternate, so
// the epilogue of one tile runs under the MMAs of the next; the scales use the
// columns behind them.
//
// Warps: 0 loads, 1 issues MMAs (even CTA), 2 owns the tensor memory, 4-19 run
// the epilogue.  Every wait is bounded: a wait that gives up raises the error
// word and the pair drains.
#include <atomic>

#include "mx_common.cuh"
#include "tc_ptx.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 640;
constexpr int kEpilogueWarps = 16;
constexpr int kMaxNt = 192;        // activation rows per tile
constexpr uint32_t kStepBytes = 128;  // bytes of a row per stage: 256 values
constexpr uint32_t kAccCols = kMaxNt;
constexpr uint32_t kScaleCol = 2 * kAccCols;

template <int kFmt, typename T> struct MxCfg {
  static constexpr int kGroups = kFmt == SCMP_MXFP4 ? 2 : 4;  // scale atoms per stage and row group
  static constexpr uint32_t kW = 128 * kStepBytes;            // a CTA's weight rows
  static constexpr uint32_t kX = kMaxNt / 2 * kStepBytes;     // a CTA's activation rows
  static constexpr uint32_t kWs = kGroups * 512;
  static constexpr uint32_t kXs = 2 * kGroups * 512;  // a tile's rows touch two row groups at most
  static constexpr uint32_t kStage = kW + kX + kWs + kXs;
  static constexpr uint32_t kScaleCols = kGroups * 4 + kGroups * 8;
  // 16-bit outputs are stored through pieces of 32 rows x 32 features, one per
  // epilogue warp
  static constexpr uint32_t kPiece = sizeof(T) == 2 ? 2048 : 0;
  static constexpr uint32_t kOut = kEpilogueWarps * kPiece;
  static constexpr int kStages = kFmt == SCMP_NVFP4 && sizeof(T) == 2 ? 5 : 6;
  static constexpr size_t kSmem = (size_t)kStages * kStage + kOut + 1024 /*align*/ + 256;
  static_assert(kStage % 1024 == 0, "swizzle atoms stay aligned");
  static_assert(kScaleCol + 2 * kScaleCols <= 512, "two sets of scales behind the accumulators");
  static_assert(kSmem <= 227 * 1024, "shared memory per CTA");
};

struct MxTiles {
  MxProduct p;
  int nt;                  // activation rows per tile (16, 32, 64, 128 or 192)
  int xrows;               // row groups (of 128) that their scales touch: 1 or 2
  uint32_t tiles_f, tiles;  // weight tiles (256 rows); all tiles, weight tiles fastest
  int steps;               // stages per tile
  int mmas;                // 64-value MMAs per tile
  bool tma_out;            // 16-bit rows of whole 16-byte pieces: stored by TMA
  bool words;              // else: 16-bit outputs are stored two features at a time
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
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// Arrival on a barrier of the pair's even CTA.  What it reports, loads of tensor
// memory that have returned, needs no release beyond the tcgen05 fence in front
// of it; a cluster-scope release waits for the warp's stores (a warp that stores
// lost 1500 cycles a tile to it).
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok));
  return ok != 0;
}
// Bounded wait of a whole warp: its lanes go on, or give up, together.  The abort
// word, the clock and the limit (a global load) are looked at after a run of
// tries only: looked at after every try they held each handover back by up to
// half a microsecond (8192^3: 207 us, now 201).
__device__ __forceinline__ bool warp_wait_cl(uint64_t *bar, uint32_t parity, volatile int *abort) {
  if (__all_sync(~0u, mbar_try_wait_cl(bar, parity))) return true;
  const unsigned long long t0 = now_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (__all_sync(~0u, mbar_try_wait_cl(bar, parity))) return true;
    bool go_on = !*abort;
    if (go_on && now_ns() - t0 > wait_limit()) {
      *abort = 1;
      go_on = false;
    }
    if (!__all_sync(~0u, go_on)) return false;
  }
}
// TMA loads into this CTA's shared memory that complete on a barrier of the
// pair's even CTA.
__device__ __forceinline__ void tma_pair_2d(uint32_t dst, const CUtensorMap *map, int x, int y,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_pair_3d(uint32_t dst, const CUtensorMap *map, int x, int y,
                                            int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// A bulk group of one TMA store (of this thread).
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, int x, int y, uint32_t src) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n"
      "cp.async.bulk.commit_group;" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(x), "r"(y), "r"(src)
      : "memory");
}

// One row of 32 neighbouring features per lane, 32 activation rows in v: scaled,
// with the bias, rounded, stored.  16-bit outputs whose pairs of features are
// words (`words`: N even, out 4-byte aligned) go out as such: neighbouring lanes
// exchange a value, so that each stores two features of one of two rows.
template <typename T, bool kFull>
__device__ __forceinline__ void store_chunk(const MxProduct &p, bool words,
                                            const uint32_t (&v)[32], float bias, int64_t row,
                                            int64_t f, int rows, int lane) {
  bool done = false;
  if constexpr (sizeof(T) == 2) if (words) {
    done = true;
    const int odd = lane & 1;
    const bool live = (f & ~(int64_t)1) < p.N;
    uint32_t *out = reinterpret_cast<uint32_t *>(static_cast<T *>(p.out) + (row + odd) * p.N +
                                                 (f & ~(int64_t)1));
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const float a = __fmaf_rn(__uint_as_float(v[j]), p.alpha, bias);
      const float b = __fmaf_rn(__uint_as_float(v[j + 1]), p.alpha, bias);
      const float other = __shfl_xor_sync(~0u, odd ? a : b, 1);
      if (live && (kFull || j + odd < rows))
        *out = odd ? pack2<T>(other, b) : pack2<T>(a, other);
      out += p.N;  // two rows of N / 2 words
    }
  }
  if (!done) {
    T *out = static_cast<T *>(p.out) + row * p.N + f;
    const bool live = f < p.N;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      if (live && (kFull || j < rows))
        *out = from_f32<T>(__fmaf_rn(__uint_as_float(v[j]), p.alpha, bias));
      out += p.N;
    }
  }
}

template <int kFmt, typename T>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    mx_pair_kernel(const __grid_constant__ MxTiles t, const __grid_constant__ CUtensorMap wmap,
                   const __grid_constant__ CUtensorMap xmap,
                   const __grid_constant__ CUtensorMap wsmap,
                   const __grid_constant__ CUtensorMap xsmap,
                   const __grid_constant__ CUtensorMap omap) {
  using Cfg = MxCfg<kFmt, T>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full =
      reinterpret_cast<uint64_t *>(smem + Cfg::kStages * Cfg::kStage + Cfg::kOut);
  uint64_t *empty = full + Cfg::kStages;
  uint64_t *tfull = empty + Cfg::kStages, *tempty = tfull + 2, *drain = tempty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(&full[s], 1);   // even CTA: its loader, and both loaders' bytes
      mbar_init(&empty[s], 1);  // commit of the MMAs that read the stage
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], kEpilogueWarps);  // even CTA: the accumulator's readers in both CTAs
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
  // All of the above may run while the kernel in front of this one in the stream
  // ends; global memory is touched from here on only.
  grid_dependency_wait();
  const uint32_t cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  const uint32_t smem0 = smem_u32(smem);

  if (warp == 0) {
    // -------------------------------------------------------------- loader
    // (the whole warp walks the stages, one elected lane issues: see the MMA warp)
    const uint32_t bars = mapa_shared(smem_u32(full), 0);
    // bytes of a stage over both CTAs; what lies past an operand's end arrives
    // as zeros and counts too
    const uint32_t bytes = 2 * (Cfg::kW + (uint32_t)t.nt / 2 * kStepBytes + Cfg::kWs +
                                (uint32_t)t.xrows * Cfg::kGroups * 512);
    int stage = 0;
    uint32_t phase = 0, issued = 0;
    bool ok = __all_sync(~0u, producers_released(abort));
    for (uint32_t tile = cluster; tile < t.tiles && ok; tile += clusters) {
      const int f0 = (int)(tile % t.tiles_f * 256 + rank * 128);
      const int n0 = (int)(tile / t.tiles_f) * t.nt, half = n0 + (int)rank * (t.nt / 2);
      for (int kb = 0; kb < t.steps; ++kb) {
        ok = warp_wait_cl(&empty[stage], phase ^ 1, abort);
        if (!ok) break;
        const uint32_t at = smem0 + stage * Cfg::kStage, bar = bars + 8u * (uint32_t)stage;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], bytes);
          tma_pair_2d(at, &wmap, kb * (int)kStepBytes, f0, bar);
          tma_pair_2d(at + Cfg::kW, &xmap, kb * (int)kStepBytes, half, bar);
          tma_pair_3d(at + Cfg::kW + Cfg::kX, &wsmap, 0, kb * Cfg::kGroups, f0 >> 7, bar);
          tma_pair_3d(at + Cfg::kW + Cfg::kX + Cfg::kWs, &xsmap, 0, kb * Cfg::kGroups, n0 >> 7,
                      bar);
        }
        __syncwarp();
        ++issued;
        if (++stage == Cfg::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // No CTA ends with copies in flight.  The even CTA sees every stage's bytes
    // arrive, and the odd one leaves after it (cluster barrier below).  When a
    // wait gave up, the odd CTA may have started copies for a stage that the
    // even one did not: it lets them land first (they take microseconds).
    if (rank == 0) {
      for (uint32_t i = issued > Cfg::kStages ? issued - Cfg::kStages : 0; i < issued; ++i)
        mbar_wait_own(&full[i % Cfg::kStages], i / Cfg::kStages & 1);
    } else if (!ok) {
      const unsigned long long t0 = now_ns();
      while (now_ns() - t0 < 2000000ull) {
      }
    }
  } else if (warp == 1 && rank == 0) {
    // --------------------------------------------------------- MMA issuer
    // the whole warp walks the stages and one elected lane issues: loop state
    // and descriptors stay warp-uniform, and so does what the instructions read
    int stage = 0;
    uint32_t phase = 0, it = 0, set = 0;
    const uint64_t desc0 = smem_desc_sw128(smem0);
    const uint64_t sdesc0 = scale_desc(smem0 + Cfg::kW + Cfg::kX);
    const uint32_t id0 = idesc<kFmt>(t.nt, 0), id2 = idesc<kFmt>(t.nt, 2);
    const bool two = t.xrows > 1;
    bool ok = true;
    for (uint32_t tile = cluster; tile < t.tiles && ok; tile += clusters, ++it) {
      const uint32_t n0 = (uint32_t)(tile / t.tiles_f) * (uint32_t)t.nt;
      const uint32_t buf = it & 1;
      if (it >= 2) ok = warp_wait_cl(&tempty[buf], ((it >> 1) - 1) & 1, abort);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * kAccCols;
      int left = t.mmas;
      for (int kb = 0; kb < t.steps; ++kb, left -= 4, set ^= 1) {
        ok = warp_wait_cl(&full[stage], phase, abort);
        if (!ok) break;
        tc_fence_after();
        // the scales of consecutive stages use two sets of columns in turn
        const uint32_t sw = tmem + kScaleCol + set * Cfg::kScaleCols, sx = sw + Cfg::kGroups * 4;
        const uint64_t d = desc_add(desc0, (uint32_t)stage * Cfg::kStage);
        const uint64_t ds = desc_add(sdesc0, (uint32_t)stage * Cfg::kStage);
        const uint32_t sxo = sx + (n0 & 127u) / 32;
        if (elect_one()) {
#pragma unroll
          for (int g = 0; g < Cfg::kGroups; ++g) {
            copy_scales(sw + g * 4, desc_add(ds, g * 512));
            copy_scales(sx + g * 8, desc_add(ds, Cfg::kWs + g * 512));
            if (two)
              copy_scales(sx + g * 8 + 4, desc_add(ds, Cfg::kWs + (Cfg::kGroups + g) * 512));
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if (kk >= left) break;  // past K
            const int g = kFmt == SCMP_MXFP4 ? kk >> 1 : kk;
            mma_pair<kFmt>(acc, desc_add(d, kk * 32), desc_add(d, Cfg::kW + kk * 32),
                           kFmt == SCMP_MXFP4 && (kk & 1) ? id2 : id0, sw + g * 4, sxo + g * 8,
                           (kb > 0 || kk > 0) ? 1u : 0u);
          }
          tc_commit_pair_both(&empty[stage]);
          if (kb == t.steps - 1) tc_commit_pair_both(&tfull[buf]);
        }
        __syncwarp();
        if (++stage == Cfg::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (elect_one()) {
      tc_commit_pair_local(drain);
      mbar_wait_own_cl(drain, 0);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    // Eight warps per accumulator (two per 32 lanes, 32-column pieces in turn), so
    // that the tiles of the two accumulators are read and stored side by side.  An
    // accumulator's next tile waits for the last load from it: two pieces are
    // loaded at once, one is stored to make room, the third is loaded and the
    // accumulator handed back before the others are stored (after two stores: 42
    // us for fc1 of 64 images in bf16, now 41).
    const uint32_t buf = (uint32_t)(warp - 4) >> 3;
    const uint32_t acc = tmem + ((uint32_t)((warp & 3) * 32) << 16) + buf * kAccCols;
    const uint32_t to = mapa_shared(smem_u32(&tempty[buf]), 0);
    const int first = ((warp - 4) >> 2 & 1) * 32;
    uint32_t turn = 0;
    for (uint32_t tile = cluster + buf * clusters; tile < t.tiles; tile += 2 * clusters, ++turn) {
      const int64_t f = (int64_t)(tile % t.tiles_f) * 256 + rank * 128 + (warp & 3) * 32 + lane;
      const int64_t n0 = (int64_t)(tile / t.tiles_f) * t.nt;
      const float bias = t.p.bias && f < t.p.N ? load_as_f32(t.p.bias, t.p.bias_dtype, f) : 0.0f;
      const int64_t left = t.p.M - n0;
      const int rows = left < t.nt ? (int)left : t.nt;
      const int f0 = (int)(f - lane);
      if (!warp_wait_cl(&tfull[buf], turn & 1, abort)) break;
      tc_fence_after();
      const auto hand_back = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_remote(to);
      };
      const auto store = [&](int j0, const uint32_t (&v)[32]) {
        if (j0 >= rows || f0 >= t.p.N) return;
        if (sizeof(T) == 2 && t.tma_out) {
          // through shared memory; a TMA store clips what lies past M and N
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
          uint16_t *piece = reinterpret_cast<uint16_t *>(smem + Cfg::kStages * Cfg::kStage +
                                                         (warp - 4) * Cfg::kPiece);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            uint32_t two = 0;
            if constexpr (sizeof(T) == 2)
              two = pack2<T>(__fmaf_rn(__uint_as_float(v[j]), t.p.alpha, bias),
                             __fmaf_rn(__uint_as_float(v[j + 1]), t.p.alpha, bias));
            piece[j * 32 + lane] = (uint16_t)two;
            piece[(j + 1) * 32 + lane] = (uint16_t)(two >> 16);
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) tma_store_2d(&omap, f0, (int)n0 + j0, smem_u32(piece));
        } else if (j0 + 32 <= rows) {
          store_chunk<T, true>(t.p, t.words, v, bias, n0 + j0, f, 32, lane);
        } else {
          store_chunk<T, false>(t.p, t.words, v, bias, n0 + j0, f, rows - j0, lane);
        }
      };
      const bool third = first + 128 < t.nt;
      uint32_t v[2][32];
      if (first < t.nt) tmem_ld32(acc + first, v[0]);
      if (first + 64 < t.nt) tmem_ld32(acc + first + 64, v[1]);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (!third) hand_back();
      store(first, v[0]);
      if (third) {
        tmem_ld32(acc + first + 128, v[0]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        hand_back();
      }
      store(first + 64, v[1]);
      if (third) store(first + 128, v[0]);
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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

// Scale atoms [row groups][groups][512 bytes] in boxes of `box_groups` x `box_rows`.
bool encode_scales(CUtensorMap *map, const uint8_t *scales, int64_t rows, int64_t groups,
                   uint32_t box_groups, uint32_t box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  cuuint64_t gdim[3] = {128, (cuuint64_t)groups, (cuuint64_t)((rows + 127) / 128)};
  cuuint64_t gstride[2] = {512, (cuuint64_t)groups * 512};
  cuuint32_t box[3] = {128, box_groups, box_rows};
  cuuint32_t estride[3] = {1u, 1u, 1u};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, const_cast<uint8_t *>(scales), gdim, gstride,
             box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 16-bit outputs in pieces of 32 rows x 32 features.
bool encode_out(CUtensorMap *map, void *out, int64_t rows, int64_t features) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  cuuint64_t gdim[2] = {(cuuint64_t)features, (cuuint64_t)rows};
  cuuint64_t gstride[1] = {(cuuint64_t)features * 2};
  cuuint32_t box[2] = {32, 32};
  cuuint32_t estride[2] = {1u, 1u};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, out, gdim, gstride, box, estride,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
cudaError_t launch(MxTiles t, int64_t kp, int64_t groups, cudaStream_t s) {
  using Cfg = MxCfg<kFmt, T>;
  auto kern = mx_pair_kernel<kFmt, T>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  // (an attribute of the function in the current context, so set in every call)
  if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)Cfg::kSmem)) != cudaSuccess)
    return e;
  // one cluster per resident pair slot (persistent tiles)
  static std::atomic<int> max_clusters[kMaxCachedDevices];
  int clusters = dev < kMaxCachedDevices ? max_clusters[dev].load(std::memory_order_relaxed) : 0;
  if (clusters <= 0) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = Cfg::kSmem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if ((e = cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg)) != cudaSuccess) return e;
    if (clusters <= 0) return cudaErrorInvalidConfiguration;
    if (dev < kMaxCachedDevices) max_clusters[dev].store(clusters, std::memory_order_relaxed);
  }
  const MxTilePlan plan = mx_tile_plan(t.p.M, t.p.N, clusters);
  t.tiles_f = plan.tiles_f;
  t.nt = plan.nt;
  t.tiles = plan.tiles;
  t.steps = (int)((kp + 255) / 256);
  t.mmas = (int)((kp + 63) / 64);
  t.xrows = t.nt > 128 ? 2 : 1;
  t.words = t.p.N % 2 == 0 && (reinterpret_cast<uintptr_t>(t.p.out) & 3) == 0;
  t.tma_out = sizeof(T) == 2 && t.p.N % 8 == 0 &&
              (reinterpret_cast<uintptr_t>(t.p.out) & 15) == 0;
  CUtensorMap wmap, xmap, wsmap, xsmap, omap = {};
  if (!encode_rows(&wmap, t.p.b, t.p.N, kp / 2, 128) ||
      !encode_rows(&xmap, t.p.a, t.p.M, kp / 2, (uint32_t)t.nt / 2) ||
      !encode_scales(&wsmap, t.p.b_scales, t.p.N, groups, Cfg::kGroups, 1) ||
      !encode_scales(&xsmap, t.p.a_scales, t.p.M, groups, Cfg::kGroups, (uint32_t)t.xrows) ||
      (t.tma_out && !encode_out(&omap, t.p.out, t.p.M, t.p.N)))
    return cudaErrorInvalidValue;
  const unsigned grid = t.tiles < (uint32_t)clusters ? t.tiles : (unsigned)clusters;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * grid, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = s;
  cfg.attrs = early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, t, wmap, xmap, wsmap, xsmap, omap);
}

template <int kFmt>
cudaError_t launch_typed(const MxTiles &t, int64_t kp, int64_t groups, cudaStream_t s) {
  if (t.p.out_dtype == SCMP_F32) return launch<kFmt, float>(t, kp, groups, s);
  if (t.p.out_dtype == SCMP_BF16) return launch<kFmt, __nv_bfloat16>(t, kp, groups, s);
  return launch<kFmt, __half>(t, kp, groups, s);
}

}  // namespace

MxTilePlan mx_tile_plan(int64_t M, int64_t N, int pairs) {
  MxTilePlan plan;
  plan.tiles_f = (uint32_t)((N + 255) / 256);
  plan.nt = tile_rows(M, plan.tiles_f, pairs);
  // (2^31 tiles of 256 x 64 outputs do not fit the memory)
  plan.tiles = plan.tiles_f * (uint32_t)((M + plan.nt - 1) / plan.nt);
  return plan;
}

cudaError_t launch_mx_matmul(const MxProduct &p, unsigned int *error, cudaStream_t s) {
  const MxLayout l = mx_layout(p.M, p.K, p.fmt);
  MxTiles t{};
  t.p = p;
  t.error = error;
  return p.fmt == SCMP_MXFP4 ? launch_typed<SCMP_MXFP4>(t, l.kp, l.groups, s)
                             : launch_typed<SCMP_NVFP4>(t, l.kp, l.groups, s);
}

cudaError_t mx_set_wait_limit(unsigned long long ns) {
  return cudaMemcpyToSymbol(g_wait_limit_ns, &ns, sizeof(ns));
}
cudaError_t mx_hold_producers(int on) {
  return cudaMemcpyToSymbol(g_hold_producers, &on, sizeof(on));
}

}  // namespace scmp
