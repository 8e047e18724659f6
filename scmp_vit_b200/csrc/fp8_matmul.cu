// Product of two operands of 8-bit floating point with a scale per block of 128,
// on the tensor cores:
//   out[m, n] = sum_b 2^(ea[m, b] + eb[n, b]) sum_{k in b} A[m, k] B[n, k] (+ bias[n]),
// A [M, K] and B [N, K] both in the layout of fp8_common.cuh.
//
// tcgen05.mma kind::mxf8f6f4 on CTA pairs (cta_group::2), which takes one e8m0
// scale per 32 values of K: the four MMAs of a block of 128 read the same byte of
// the scale word, and an atom of scales serves four blocks.  The accumulator is
// never scaled by the CUDA cores, so the epilogue runs once per tile.  256 rows of
// B are the accumulator's lanes (128 per CTA), rows of A its columns: a lane owns
// one output feature and 32 lanes store 32 neighbouring outputs.  A stage is two
// blocks of K: both operands' codes (128-byte rows, 128-byte swizzle) by TMA,
// completing on the even CTA's barrier; every other one brings the scales too.  (With
// one block per stage the issuing warp, some 450 cycles of waits and descriptors a
// stage, held a block to 270 ns at every width; with two 240 at 192 columns, 183 at
// 128, 160 at 64, at full clocks.)
//
// Tensor memory holds an accumulator of 256 columns, one of 192 and the scales, so
// that the epilogue of a tile runs under the MMAs of the next, and a pair takes its
// tiles 256 and 192 rows of A wide in turn: fewer bytes per product than 192 alone.
// Where that leaves pairs idle, tiles have one width (plan_of).
//
// Long sums are bound by power (8192^3: 410 us at 1.1 GHz, 343 of zeros at 1.97), fc1 of 64
// images ([16448, 1024] by [4096, 1024], bf16: 62 us) by its outputs besides: without
// their stores it takes 47.  At K = 128, which leaves little but the stores, pieces of
// 64-byte rows take 33 us, of 128-byte rows 38, from registers 42: what these stores cost
// beside these loads, not what an SM can write (the dequantiser's fp32 leave at 17
// bytes a clock and SM, 33 us are 14).  One stage of B for both accumulators
// loads 27 % less, but then their tiles end together: fc1 63 us, K = 4096 186 for 193.
//
// Where a sum is so long that the bits that the tensor core cuts off would show, it is
// made in pieces (kPieces, kWholeBlocks).
//
// Warps: 0 loads, 1 issues MMAs (even CTA), 2 owns the tensor memory, 4-19 run
// the epilogue.  Every wait is bounded: a wait that gives up raises the error
// word and the pair drains.
#include <atomic>

#include "fp8_common.cuh"
#include "mx_pair.cuh"
#include "tc_ptx.cuh"

namespace scmp {
namespace {

constexpr int kThreads = 640;
constexpr int kEpilogueWarps = 16;
constexpr int kWide = 256, kNarrow = 192;  // rows of A: the accumulators' columns
constexpr int kPerStage = 2;               // blocks of K per stage
constexpr int kStages = 3;
constexpr int kPieceCols = 128;            // of a sum in pieces, at most
constexpr uint32_t kScaleCol = kWide + kNarrow;
constexpr uint32_t kScaleCols = 4 + 12;  // of an atom of B, three of A

constexpr uint32_t kW = 128 * kRowBytes;        // a CTA's rows of B, one block of K
constexpr uint32_t kX = kWide / 2 * kRowBytes;  // a CTA's rows of A, at most
constexpr uint32_t kStage = kPerStage * (kW + kX);
constexpr uint32_t kScales = 4 * 512;  // one row group of B, up to three of A
constexpr uint32_t kScalesAt = kStages * kStage;
// 16-bit outputs are stored through pieces of 16 rows x 32 features, one per epilogue
// warp (of 32 rows they do not fit).
constexpr int kPieceRows = 16;
constexpr uint32_t kPiece = kPieceRows * 64;
constexpr uint32_t kOutAt = kScalesAt + kStages * kScales;
constexpr uint32_t kBarsAt = kOutAt + kEpilogueWarps * kPiece;
constexpr size_t kSmem = (size_t)kBarsAt + 1024 /*align*/ + 256;
static_assert(kStage % 1024 == 0 && kOutAt % 512 == 0 && kPiece % 512 == 0,
              "swizzle atoms stay aligned");
static_assert(kScaleCol + 2 * kScaleCols <= 512, "two sets of scales behind the accumulators");
static_assert(kSmem <= 227 * 1024, "shared memory per CTA");

struct Fp8Tiles {
  Fp8Product p;
  Fp8TilePlan plan;
  uint32_t group, group_units;  // tiles of B's rows that are walked together; their units
  int xrows;               // row groups (of 128) that a tile's scales of A touch, at most
  int block0, blocks;      // blocks of K of this launch
  int steps;               // stages per tile
  int piece;               // stages per piece of a sum in pieces
  bool tma_out;            // 16-bit rows of whole 16-byte pieces: stored by TMA
  bool words;              // else: 16-bit outputs are stored two features at a time
  bool add;                // fp32 outputs: added to what is there
  unsigned int *error;
};

// The tiles of a pair in order: f(first row of B, first row of A, which width,
// accumulator) until it is false.
template <typename F>
__device__ __forceinline__ void for_tiles(const Fp8Tiles &t, F &&f) {
  const uint32_t clusters = gridDim.x >> 1;
  uint32_t it = 0;
  for (uint32_t u = blockIdx.x >> 1; u < t.plan.units; u += clusters) {
    uint32_t begin = 0, width = t.group, at = u;
    if (width < t.plan.tiles_f) {
      const uint32_t group = u / t.group_units;
      begin = group * width;
      at -= group * t.group_units;
      if (t.plan.tiles_f - begin < width) width = t.plan.tiles_f - begin;
    }
    const uint32_t q = at / width;
    const int f0 = (int)(begin + at - q * width) * 256;
    int64_t n0 = (int64_t)q * (t.plan.w[0] + t.plan.w[1]);
    for (int sub = 0; sub < 2; ++sub) {
      if (t.plan.w[sub] == 0 || n0 >= t.p.M) break;
      const uint32_t buf = t.plan.w[1] ? (uint32_t)sub : t.plan.w[0] > kNarrow ? 0u : it & 1u;
      ++it;
      if (!f(f0, (int)n0, sub, buf)) return;
      n0 += t.plan.w[0];
    }
  }
}

// (of an MMA n columns wide; A and B e4m3: 0)
__host__ __device__ constexpr uint32_t idesc(int n) {
  return ((uint32_t)(n >> 3) << 17)         // N
         | (1u << 23)                       // scales e8m0
         | ((uint32_t)(256 >> 4) << 24);    // M over the pair
}
// The byte of the scale words that an MMA reads.
__device__ __forceinline__ uint32_t idesc_byte(uint32_t id, uint32_t byte) {
  return id | byte << 4 | byte << 29;
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], "
      "p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb)
      : "memory");
}

// 32 lanes x 32 columns of tensor memory as fragments of 8 x 8 (lanes x columns):
// thread t holds lane t / 4 and columns 2 (t % 4), + 1 of each, in v[16 h + 4 c + 2 l]
// and the next for lanes 16 h + 8 l .. and columns 8 c ...
__device__ __forceinline__ void tmem_ld_fragments(uint32_t taddr, uint32_t (&v)[32]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t *r = v + 16 * h;
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr + ((uint32_t)(16 * h) << 16)));
  }
}
// Four 8 x 8 matrices of 16-bit values, a fragment register each, transposed into
// shared memory: thread t gives the address of row t % 8 of matrix t / 8 (16 bytes).
__device__ __forceinline__ void store_transposed(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                                 uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// kPieces: a tile's sum in pieces, each in the one or the other accumulator, which the
// epilogue's warps add up in registers, 32 of at most 128 columns each.
template <typename T, bool kPieces>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    fp8_pair_kernel(const __grid_constant__ Fp8Tiles t, const __grid_constant__ CUtensorMap wmap,
                    const __grid_constant__ CUtensorMap xmap0,
                    const __grid_constant__ CUtensorMap xmap1,
                    const __grid_constant__ CUtensorMap wsmap,
                    const __grid_constant__ CUtensorMap xsmap,
                    const __grid_constant__ CUtensorMap omap) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kBarsAt);
  uint64_t *empty = full + kStages;
  uint64_t *tfull = empty + kStages, *tempty = tfull + 2, *drain = tempty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  // one accumulator (or one at a time): all epilogue warps read it
  const bool alone = kPieces || (t.plan.w[1] == 0 && t.plan.w[0] > kNarrow);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);   // even CTA: its loader, and both loaders' bytes
      mbar_init(&empty[s], 1);  // commit of the MMAs that read the stage
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      // even CTA: the accumulator's readers in both CTAs
      mbar_init(&tempty[i], alone ? 2 * kEpilogueWarps : kEpilogueWarps);
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
  const uint32_t smem0 = smem_u32(smem);

  if (warp == 0) {
    // -------------------------------------------------------------- loader
    // (the whole warp walks the stages, one elected lane issues: see the MMA warp)
    const uint32_t bars = mapa_shared(smem_u32(full), 0);
    const uint32_t scale_bytes = 2 * (1u + (uint32_t)t.xrows) * 512;
    int stage = 0;
    uint32_t phase = 0, issued = 0;
    bool ok = __all_sync(~0u, producers_released(abort));
    if (ok) for_tiles(t, [&](int f0, int n0, int sub, uint32_t) {
      const int w = t.plan.w[sub], half = n0 + (int)rank * (w / 2);
      const CUtensorMap *xmap = sub ? &xmap1 : &xmap0;
      // bytes of a stage over both CTAs; what lies past an operand's end arrives as
      // zeros and counts too
      const uint32_t bytes = 2 * kPerStage * (kW + (uint32_t)w / 2 * kRowBytes);
      f0 += (int)rank * 128;
      for (int kb = 0; kb < t.steps; ++kb) {
        ok = warp_wait_cl(&empty[stage], phase ^ 1, abort);
        if (!ok) return false;
        const uint32_t at = smem0 + stage * kStage, bar = bars + 8u * (uint32_t)stage;
        const int block = t.block0 + kb * kPerStage;
        if (elect_one()) {
          const bool first = kb % (4 / kPerStage) == 0;  // brings four blocks' scales
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], first ? bytes + scale_bytes : bytes);
          tma_pair_3d(at, &wmap, 0, f0, block, bar);
          tma_pair_3d(at + kPerStage * kW, xmap, 0, half, block, bar);
          if (first) {
            const uint32_t sat = smem0 + kScalesAt + stage * kScales;
            tma_pair_3d(sat, &wsmap, 0, block >> 2, f0 >> 7, bar);
            tma_pair_3d(sat + 512, &xsmap, 0, block >> 2, n0 >> 7, bar);
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      return true;
    });
    // No CTA ends with copies in flight.  The even CTA sees every stage's bytes
    // arrive, and the odd one leaves after it (cluster barrier below).  When a
    // wait gave up, the odd CTA may have started copies for a stage that the
    // even one did not: it lets them land first (they take microseconds).
    if (rank == 0) {
      for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
        mbar_wait_own(&full[i % kStages], i / kStages & 1);
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
    uint32_t phase = 0, set = 0, turn = 0, uses[2] = {0, 0};
    const uint64_t desc0 = smem_desc_sw128(smem0);
    const uint64_t sdesc0 = scale_desc(smem0 + kScalesAt);
    for_tiles(t, [&](int, int n0, int sub, uint32_t of_tile) {
      const uint32_t w = (uint32_t)t.plan.w[sub], id0 = idesc((int)w);
      const uint32_t xblock = w / 2 * kRowBytes, offset = ((uint32_t)n0 & 127u) / 32;
      int kb = 0;
      do {
        const uint32_t buf = kPieces ? turn++ & 1 : of_tile;
        const uint32_t use = buf ? uses[1]++ : uses[0]++;
        if (use > 0 && !warp_wait_cl(&tempty[buf], (use - 1) & 1, abort)) return false;
        tc_fence_after();
        const uint32_t acc = tmem + buf * kWide;
        const int begin = kb, end = kPieces && kb + t.piece < t.steps ? kb + t.piece : t.steps;
        for (; kb < end; ++kb) {
          if (!warp_wait_cl(&full[stage], phase, abort)) return false;
          tc_fence_after();
          // consecutive atoms of scales use two sets of columns in turn
          const bool first = kb % (4 / kPerStage) == 0;
          if (first) set ^= 1;
          const uint32_t sw = tmem + kScaleCol + set * kScaleCols, sx = sw + 4;
          const uint64_t d = desc_add(desc0, (uint32_t)stage * kStage);
          const uint64_t dx = desc_add(d, kPerStage * kW);
          if (elect_one()) {
            if (first) {
              const uint64_t ds = desc_add(sdesc0, (uint32_t)stage * kScales);
              copy_scales(sw, ds);
              for (int i = 0; i < t.xrows; ++i)
                copy_scales(sx + 4 * i, desc_add(ds, 512 + 512 * i));
            }
#pragma unroll
            for (int b = 0; b < kPerStage; ++b) {
              if (b > 0 && kb * kPerStage + b >= t.blocks) break;  // past K
              const uint32_t id = idesc_byte(id0, (uint32_t)(kb * kPerStage + b) & 3u);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_pair(acc, desc_add(d, b * kW + kk * 32), desc_add(dx, b * xblock + kk * 32),
                         id, sw, sx + offset, (kb > begin || b > 0 || kk > 0) ? 1u : 0u);
            }
            tc_commit_pair_both(&empty[stage]);
            if (kb == end - 1) tc_commit_pair_both(&tfull[buf]);
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      } while (kPieces && kb < t.steps);
      return true;
    });
    if (elect_one()) {
      tc_commit_pair_local(drain);
      mbar_wait_own_cl(drain, 0);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    // Eight warps per accumulator (two per 32 lanes, pieces of 32 columns in turn), so
    // that the tiles of the two accumulators are read and stored side by side.  An
    // accumulator's next tile waits for the last load from it: two pieces are
    // loaded at once and stored while the next are on their way.
    //
    // 16-bit rows that a TMA store can write are loaded as 8 x 8 fragments, which go to
    // shared memory transposed, 512 bytes at a time, in the order of the store's
    // 64-byte swizzle (no conflicts; two bytes at a time they took 72 shared-memory
    // cycles a piece, which the MMAs' operands compete for).  Others go from
    // registers: a lane holds a feature.
    const bool by_tma = sizeof(T) == 2 && t.tma_out;
    const uint32_t mine = (uint32_t)(warp - 4) >> 3, half = (uint32_t)(warp - 4) >> 2 & 1;
    const int first = (int)(alone ? 2 * mine + half : half) * 32, stride = alone ? 128 : 64;
    const uint32_t piece = smem0 + kOutAt + (uint32_t)(warp - 4) * kPiece;
    uint32_t turn = 0;
    for_tiles(t, [&](int f0, int n0, int sub, uint32_t of_tile) {
      if (!alone && of_tile != mine) return true;
      f0 += (int)rank * 128 + (warp & 3) * 32;
      const auto bias_of = [&](int f) {
        return t.p.bias && f < t.p.N ? load_as_f32(t.p.bias, t.p.bias_dtype, f) : 0.0f;
      };
      float bias[4];  // of a fragment's features, or of the lane's
#pragma unroll
      for (int i = 0; i < 4; ++i) bias[i] = bias_of(f0 + (by_tma ? 8 * i + (lane >> 2) : lane));
      const int64_t left = t.p.M - n0;
      const int w = t.plan.w[sub], rows = left < w ? (int)left : w;
      uint32_t buf = kPieces ? turn & 1 : of_tile;
      if (!warp_wait_cl(&tfull[buf], (kPieces ? turn >> 1 : turn) & 1, abort)) return false;
      ++turn;
      tc_fence_after();
      uint32_t acc = tmem + ((uint32_t)((warp & 3) * 32) << 16) + buf * kWide;
      const auto hand_back = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_remote(mapa_shared(smem_u32(&tempty[buf]), 0));
      };
      const auto load = [&](int j0, uint32_t (&v)[32]) {
        if (by_tma)
          tmem_ld_fragments(acc + j0, v);
        else
          tmem_ld32(acc + j0, v);
      };
      const auto store = [&](int j0, uint32_t (&v)[32]) {
        if (j0 >= rows || f0 >= t.p.N) return;
        if constexpr (sizeof(T) == 2) if (by_tma) {
          // (a TMA store clips what lies past M and N)
#pragma unroll
          for (int h = 0; h < 32; h += kPieceRows) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
#pragma unroll
            for (int c = 0; c < kPieceRows / 8; ++c) {
              uint32_t m[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t *r = v + 16 * (i >> 1) + 4 * (h / 8 + c) + 2 * (i & 1);
                m[i] = pack2<T>(__uint_as_float(r[0]) + bias[i], __uint_as_float(r[1]) + bias[i]);
              }
              const int row = 8 * c + (lane & 7), chunk = lane >> 3;
              store_transposed(piece + row * 64 + (chunk ^ (row >> 1 & 3)) * 16, m[0], m[1], m[2],
                               m[3]);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && j0 + h < rows) tma_store_2d(&omap, f0, n0 + j0 + h, piece);
          }
          return;
        }
        const int64_t f = f0 + lane;
        if constexpr (sizeof(T) == 4) if (t.add && f < t.p.N) {
          const float *out = static_cast<const float *>(t.p.out) + (int64_t)(n0 + j0) * t.p.N + f;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j0 + j < rows) v[j] = __float_as_uint(__uint_as_float(v[j]) + out[j * t.p.N]);
        }
        if (j0 + 32 <= rows)
          store_chunk<T, true>(t.p, 1.0f, t.words, v, bias[0], n0 + j0, f, 32, lane);
        else
          store_chunk<T, false>(t.p, 1.0f, t.words, v, bias[0], n0 + j0, f, rows - j0, lane);
      };
      uint32_t v[2][32];
      if constexpr (kPieces) {
        // v[1]: the sum of the pieces so far
#pragma unroll
        for (int j = 0; j < 32; ++j) v[1][j] = 0;
#pragma unroll 1
        for (int kb = 0;;) {
          if (first < w) {
            load(first, v[0]);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int j = 0; j < 32; ++j)
              v[1][j] = __float_as_uint(__uint_as_float(v[1][j]) + __uint_as_float(v[0][j]));
          }
          hand_back();
          if ((kb += t.piece) >= t.steps) break;
          buf = turn & 1;
          if (!warp_wait_cl(&tfull[buf], turn >> 1 & 1, abort)) return false;
          ++turn;
          tc_fence_after();
          acc = tmem + ((uint32_t)((warp & 3) * 32) << 16) + buf * kWide;
        }
        if (first < w) store(first, v[1]);
        return true;
      }
      if (first >= w) hand_back();
#pragma unroll 1
      for (int j0 = first; j0 < w; j0 += 2 * stride) {
        load(j0, v[0]);
        if (j0 + stride < w) load(j0 + stride, v[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (j0 + 2 * stride >= w) hand_back();
        store(j0, v[0]);
        if (j0 + stride < w) store(j0 + stride, v[1]);
      }
      return true;
    });
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

// Codes as [blocks][rows][128 bytes], in boxes of a stage's blocks.
bool encode_blocks(CUtensorMap *map, const uint8_t *data, int64_t rows, const Fp8Layout &l,
                   uint32_t box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  cuuint64_t gdim[3] = {kRowBytes, (cuuint64_t)rows, (cuuint64_t)l.blocks};
  cuuint64_t gstride[2] = {(cuuint64_t)l.kp, kRowBytes};
  cuuint32_t box[3] = {kRowBytes, box_rows, kPerStage};
  cuuint32_t estride[3] = {1u, 1u, 1u};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(data), gdim, gstride,
             box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ns of one block of K for a tile `w` wide (measured at full clocks: 64 160, 128
// 183, 192 240; 256 by its MMAs).
double block_ns(int w) {
  const double issue = 100 + 0.65 * w, math = 1.2 * w;
  return issue > math ? issue : math;
}
// The same of a tile's part that no MMA hides.
constexpr double kTileNs = 250, kAloneNs = 2000;

// Widths: one tile for up to 32 rows (16 rows by [16384, 1024]: 6.0 us, a tile of 64
// 6.7; 32 rows 6.1 and 6.5; [4096, 4096] 9.0 and 9.1); else what costs least among 64, 128 and 192
// throughout, 256 alone, and 256 and 192 in turn, whose starts are all multiples of
// 64 rows (the scale columns they begin at are even); among 64 and 128 for a sum in
// pieces.
Fp8TilePlan plan_of(int64_t M, int64_t N, int64_t blocks, int pairs, bool pieces = false) {
  Fp8TilePlan best{};
  best.tiles_f = (uint32_t)((N + 255) / 256);
  best.units = best.tiles_f;
  if (M <= 32) {
    best.w[0] = M <= 16 ? 16 : 32;
    return best;
  }
  constexpr int kWidths[5][2] = {{kWide, kNarrow}, {kNarrow, 0}, {128, 0}, {64, 0}, {kWide, 0}};
  double best_ns = 0;
  for (const auto &w : kWidths) {
    if (pieces && w[0] > kPieceCols) continue;
    const int pitch = w[0] + w[1];
    const int64_t units = best.tiles_f * ((M + pitch - 1) / pitch);
    double ns = blocks * block_ns(w[0]) + (w[0] > kNarrow && !w[1] ? kAloneNs : kTileNs);
    if (w[1]) ns += blocks * block_ns(w[1]) + kTileNs;
    ns *= (double)((units + pairs - 1) / pairs);
    if (best.w[0] == 0 || ns < best_ns) {
      best_ns = ns;
      best.w[0] = w[0];
      best.w[1] = w[1];
      // (2^31 tiles of 256 x 64 outputs do not fit the memory)
      best.units = (uint32_t)units;
    }
  }
  return best;
}

// Long sums.  An MMA cuts each of its 32 products off at 2^-25 of the power of two of
// the largest term (the running sum is one) and what comes out at 2^-23: at most 9 * 2^-23
// of the running sum per 32 values, all in one direction where all products have one
// sign.  Positive values over many powers of two (e^(2 z), z normal) lose 0.4 * 2^-23 per
// 32 on average over 4096 of them (6e-6 of the sum, 3e-5 at most), 0.6 over 16384, 1 over
// 524288; normal values of both signs a root mean square of 5e-7 of the outputs' over
// 4096 and 3e-6 over 16384 (rounded 1e-7).
//
// fp32 outputs of more than kSumBlocks go in launches of at most so many that add up
// in the outputs.  16-bit outputs go in one launch, and in pieces of kPieceBlocks that
// the epilogue adds up, rounded, from where the cut bits would come near the type's
// half step (2.4e-4 to 4.9e-4 for fp16): above 16384 values for fp16 (4e-5 on average in
// the case above), eight times that for bf16.  In fp16 that case is 2e-4 off on average
// over 65536 in one piece and 2e-3 over 524288, in pieces 3e-6 and 1e-6.  Narrower tiles
// cost time: fp16 1024 rows by [4096, 16512] 71 us (in one piece 53), 4096 by [4096, 32768]
// 533 (474).
constexpr int64_t kSumBlocks = 32;
constexpr int64_t kPieceBlocks = 8;
template <typename T> constexpr int64_t kWholeBlocks = __is_same(T, __half) ? 128 : 1024;
static_assert(kPieceBlocks % 4 == 0, "a piece begins with an atom of scales");

template <typename T, bool kPieces>
cudaError_t launch(Fp8Tiles t, const Fp8Layout &l, cudaStream_t s) {
  auto kern = fp8_pair_kernel<T, kPieces>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  // (an attribute of the function in the current context, so set in every call)
  if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem)) !=
      cudaSuccess)
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
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if ((e = cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg)) != cudaSuccess) return e;
    if (clusters <= 0) return cudaErrorInvalidConfiguration;
    if (dev < kMaxCachedDevices) max_clusters[dev].store(clusters, std::memory_order_relaxed);
  }
  const int64_t launches =
      sizeof(T) == 4 ? (l.blocks + kSumBlocks - 1) / kSumBlocks : 1;
  const int64_t share = ((l.blocks + launches - 1) / launches + 3) / 4 * 4;  // whole scale atoms
  t.plan = plan_of(t.p.M, t.p.N, launches > 1 ? share : l.blocks, clusters, kPieces);
  const int *w = t.plan.w;
  t.piece = (int)kPieceBlocks / kPerStage;
  t.xrows = w[0] > kNarrow ? 3 : w[0] > 128 ? 2 : 1;
  t.words = t.p.N % 2 == 0 && (reinterpret_cast<uintptr_t>(t.p.out) & 3) == 0;
  t.tma_out = sizeof(T) == 2 && t.p.N % 8 == 0 &&
              (reinterpret_cast<uintptr_t>(t.p.out) & 15) == 0;
  CUtensorMap wmap, xmap0, xmap1 = {}, wsmap, xsmap, omap = {};
  if (!encode_blocks(&wmap, t.p.b, t.p.N, l, 128) ||
      !encode_blocks(&xmap0, t.p.a, t.p.M, l, (uint32_t)w[0] / 2) ||
      (w[1] && !encode_blocks(&xmap1, t.p.a, t.p.M, l, (uint32_t)w[1] / 2)) ||
      !encode_scales(&wsmap, t.p.b_scales, t.p.N, l.groups, 1, 1) ||
      !encode_scales(&xsmap, t.p.a_scales, t.p.M, l.groups, 1, (uint32_t)t.xrows) ||
      (t.tma_out && !encode_out(&omap, t.p.out, t.p.M, t.p.N, kPieceRows,
                                 CU_TENSOR_MAP_SWIZZLE_64B)))
    return cudaErrorInvalidValue;
  // As many tiles of B's rows at a time as stay in L2 beside what streams past them
  // (16 MB), unless all of them do.  In groups / not: 8192^3 410 / 438 us, 8192 x 8192 x
  // 4096 211 / 236, 2048 rows by [8192, 8192] 108 / 114, 4096 by [8192, 4096] 110 / 106.
  const int64_t bytes = 256 * l.kp;
  t.group = t.plan.tiles_f;
  if (t.plan.tiles_f * bytes > (24 << 20))
    t.group = bytes < (16 << 20) ? (uint32_t)((16 << 20) / bytes) : 1u;
  t.group_units = t.group * (t.plan.units / t.plan.tiles_f);
  const unsigned grid = t.plan.units < (uint32_t)clusters ? t.plan.units : (unsigned)clusters;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * grid, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cfg.attrs = early;
  cfg.numAttrs = 1;
  for (int64_t block = 0; block < l.blocks; block += share) {
    t.block0 = (int)block;
    t.blocks = (int)(l.blocks - block < share || launches == 1 ? l.blocks - block : share);
    t.steps = (t.blocks + kPerStage - 1) / kPerStage;
    t.add = block > 0;
    if (t.add) t.p.bias = nullptr;
    if ((e = cudaLaunchKernelEx(&cfg, kern, t, wmap, xmap0, xmap1, wsmap, xsmap, omap)) !=
        cudaSuccess)
      return e;
    add_launches(1);
    if (launches == 1) break;
  }
  return cudaSuccess;
}

template <typename T> cudaError_t launch_16(const Fp8Tiles &t, const Fp8Layout &l, cudaStream_t s) {
  return l.blocks > kWholeBlocks<T> ? launch<T, true>(t, l, s) : launch<T, false>(t, l, s);
}

}  // namespace

Fp8TilePlan fp8_tile_plan(int64_t M, int64_t N, int64_t K, int pairs) {
  return plan_of(M, N, (K + kFp8Block - 1) / kFp8Block, pairs);
}

cudaError_t launch_fp8_matmul(const Fp8Product &p, unsigned int *error, cudaStream_t s) {
  const Fp8Layout l = fp8_layout(p.M, p.K);
  Fp8Tiles t{};
  t.p = p;
  t.error = error;
  if (p.out_dtype == SCMP_F32) return launch<float, false>(t, l, s);
  if (p.out_dtype == SCMP_BF16) return launch_16<__nv_bfloat16>(t, l, s);
  return launch_16<__half>(t, l, s);
}

cudaError_t fp8_set_wait_limit(unsigned long long ns) {
  return cudaMemcpyToSymbol(g_wait_limit_ns, &ns, sizeof(ns));
}
cudaError_t fp8_hold_producers(int on) {
  return cudaMemcpyToSymbol(g_hold_producers, &on, sizeof(on));
}

}  // namespace scmp
