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
  float *part;  // inverse: [blocks of q, then of k][2][D] partial sums, nullable
  // set by the launcher: lanes per head row; heads per thread of a unit; units per
  // token block, of q, of q and k, of all; backward: blocks of q, of q and k, of all
  int lanes, heads_per, units_q, units_qk, units_all;
  uint32_t token_blocks, blocks_q, blocks_qk, blocks_all;
};
// Partial sums of a backward pass: blocks of q and of q and k.
struct QkNormBlocks {
  uint32_t q, qk, all;
};
QkNormBlocks qknorm_bwd_blocks(int64_t H, int64_t Hk);

cudaError_t launch_qknorm(const QkNormParams &p, int dtype, cudaStream_t s);
// grads: of q's weight and bias, k's weight and bias (each nullable).
cudaError_t launch_qknorm_sum(const QkNormParams &p, void *const (&grads)[4], cudaStream_t s);

}  // namespace scmp
