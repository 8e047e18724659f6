// Pieces of the block-scaled products on CTA pairs (4-bit and 8-bit): scale copies,
// waits, loads and stores of the pair, tensor maps.  Internal linkage.
#pragma once

#include "mx_common.cuh"
#include "tc_ptx.cuh"

namespace scmp {
namespace {

constexpr uint32_t kRowBytes = 128;  // bytes of an operand's row per stage

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

// One row of 32 neighbouring features per lane, 32 activation rows in v: scaled by
// alpha, with the bias, rounded, stored to p.out (rows of p.N).  16-bit outputs whose pairs of features are
// words (`words`: N even, out 4-byte aligned) go out as such: neighbouring lanes
// exchange a value, so that each stores two features of one of two rows.
template <typename T, bool kFull, typename P>
__device__ __forceinline__ void store_chunk(const P &p, float alpha, bool words,
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
      const float a = __fmaf_rn(__uint_as_float(v[j]), alpha, bias);
      const float b = __fmaf_rn(__uint_as_float(v[j + 1]), alpha, bias);
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
        *out = from_f32<T>(__fmaf_rn(__uint_as_float(v[j]), alpha, bias));
      out += p.N;
    }
  }
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

// 16-bit outputs in pieces of 32 features.
bool encode_out(CUtensorMap *map, void *out, int64_t rows, int64_t features, uint32_t box_rows,
                CUtensorMapSwizzle swizzle) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  cuuint64_t gdim[2] = {(cuuint64_t)features, (cuuint64_t)rows};
  cuuint64_t gstride[1] = {(cuuint64_t)features * 2};
  cuuint32_t box[2] = {32, box_rows};
  cuuint32_t estride[2] = {1u, 1u};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, out, gdim, gstride, box, estride,
             CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
             CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace scmp
