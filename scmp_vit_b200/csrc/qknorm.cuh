// Arguments of the qkv split with norms of queries and keys (qknorm.cu).
#pragma once

#include "rotary.cuh"

namespace scmp {

struct QkNormParams {
  RotaryParams r;  // axes 0: no positions; inverse: q, k, v are gradients, qkv the result
  const void *x;   // inverse: the forward's qkv
  const void *weight[2], *bias[2];  // of q, k: [D] of param_dtype; biases nullable
  int param_dtype;
  float eps;
  bool rms;
  float *part;     // inverse: [blocks][q, k][weight, bias][D] partial sums, nullable
  void *grads[4];  // with part: of q's weight and bias, k's weight and bias, each nullable
  // set by the launcher: whether the lanes of a token hold exactly D elements; lanes
  // per token; heads of a unit; units (of a token block each), token blocks by splits
  bool whole;
  int lanes, heads_per;
  uint32_t splits, units;
};
// Floats of workspace of a backward pass with gradients of parameters.
size_t qknorm_part_floats(int64_t D);
// One launch, two with part.
cudaError_t launch_qknorm(const QkNormParams &p, int dtype, cudaStream_t s);

}  // namespace scmp
