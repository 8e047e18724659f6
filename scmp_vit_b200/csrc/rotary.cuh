// Arguments of the rotary qkv split (rotary.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/scmp_b200.h"
#include "mx_common.cuh"

namespace scmp {

struct RotaryParams {
  void *qkv;         // [B, N, H + 2 Hk, D]
  void *q, *k, *v;   // [B, H, N, D], [B, Hk, N, D], and v the same or [B, Hk, D, N]
  const float2 *table;
  const int32_t *pos;  // [N, axes] or [B, N, axes]
  int64_t B, N, H, Hk;
  int D, axes;
  int dims[SCMP_MAX_AXES], sizes[SCMP_MAX_AXES];
  int64_t table_at[SCMP_MAX_AXES];  // first entry of each axis
  bool pos_batched, interleaved, v_transposed, inverse;
  // set by the launcher: pieces per head row, tokens per sample, the blocks that
  // turn heads (each a split of them) in front of the transposed tiles
  FastDiv per{1}, tokens{1};
  int heads_per;
  uint32_t splits, turn_blocks;
};
cudaError_t launch_rotary(const RotaryParams &p, int dtype, cudaStream_t s);

}  // namespace scmp
