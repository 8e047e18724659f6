// Arguments of counter-based dropout (dropout.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/scmp_b200.h"

namespace scmp {

struct DropoutParams {
  const void *x, *residual;  // residual nullable
  void *y;
  int64_t n, span;  // elements; consecutive elements that share a draw
  uint64_t seed, offset;
  const uint64_t *state;  // nullable: seed and what is added to offset, on the device
  uint64_t threshold;     // a draw below it is dropped; up to 2^32
  float scale;            // of what is kept
};
cudaError_t launch_dropout(const DropoutParams &p, int dtype, cudaStream_t s);

}  // namespace scmp
