// Arguments of counter-based dropout (dropout.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/scmp_b200.h"
#include "mx_common.cuh"

namespace scmp {

struct DropoutParams {
  const void *x, *residual;  // residual nullable
  void *y;
  int64_t n, span;  // elements; consecutive elements that share a draw
  uint64_t offset;
  const uint64_t *state;  // nullable: seed and what is added to offset, on the device
  uint32_t keys[20];      // of the generator's rounds, set by the launcher
  FastDiv per_span{1};    // span, set by the launcher
  bool none;              // nothing is dropped
  uint32_t limit;         // else: a draw up to it is
  float scale;            // of what is kept
};
// seed: not used with state
cudaError_t launch_dropout(DropoutParams p, uint64_t seed, int dtype, cudaStream_t s);

}  // namespace scmp
