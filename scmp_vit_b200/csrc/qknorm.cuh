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
  bool rms, whole;  // whole (set by the launcher): the lanes hold exactly D elements
  float *part;  // inverse: [blocks of q, then of k][2][D] partial sums, nullable
  void *grads[4];  // with part: of q's weight and bias, k's weight and bias, each nullable
  // set by the launcher: lanes per head row; heads per thread of a unit; units per
  // token block, of q, of q and k, of all; backward: blocks of q, of q and k, of all
  int lanes, heads_per, units_q, units_qk, units_all;
  uint32_t token_blocks, blocks_q, blocks_qk, blocks_all;
};
// Floats of workspace of a backward pass with gradients of parameters.
size_t qknorm_part_floats(int64_t H, int64_t Hk, int64_t D);
// One launch, two with part.
cudaError_t launch_qknorm(const QkNormParams &p, int dtype, cudaStream_t s);

}  // namespace scmp
