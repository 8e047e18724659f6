// Arguments of the gated residual + norm kernels (norm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/scmp_b200.h"
#include "mx_common.cuh"

namespace scmp {

// x, y, r [rows, C] of one type, parameters [C] (gate [groups, C]) of that type
// or fp32; null pointers leave their step out.
struct NormParams {
  const void *x, *y;
  const void *weight, *bias, *gamma, *gate, *post_weight, *post_bias;
  void *r;         // written when y is given
  void *h;         // nullable
  float2 *stats;   // nullable [2][rows]: mean and 1 / deviation of r, of y (post norm)
  uint8_t *mx_data, *mx_scales;  // nullable: h's 4-bit codes (16-byte rows only)
  int64_t rows, rows_per_gate, kp, groups;
  int C;
  float eps;
  bool rms, h_f32;
  int fmt;
  int warps_per_row;  // set by the launcher
  FastDiv per_gate{1};  // rows_per_gate
  int64_t row_end;    // rows that have output: all, or whole atoms of 4-bit scales
};

struct NormBwdParams {
  const void *r, *y, *dr, *dh;  // y, dr, dh nullable
  const void *weight, *gamma, *gate, *post_weight, *post_bias;
  const float2 *stats;
  void *dx, *dy;  // nullable
  void *dweight, *dbias, *dgamma, *dgate, *dpost_weight, *dpost_bias;  // nullable
  float *part;  // nullable (no parameter gradient wanted), see NormBwdPlan
  int64_t rows, groups;
  int C;
  bool rms;
  int64_t rows_per_group, blocks_per_group;  // set by the launcher, as below
  int warps_per_row, share;
};

struct NormBwdPlan {
  int warps_per_row, slots;  // slots: rows a block works on at a time
  int64_t blocks_per_group;
  int64_t part_floats;  // workspace
};
NormBwdPlan norm_bwd_plan(int64_t rows, int64_t groups, int64_t C);
// Floats of workspace.
int64_t norm_bwd_floats(int64_t rows, int64_t groups, int64_t C);

constexpr int64_t kNormMaxC = 8192;  // 16 warps of 16 elements per lane

cudaError_t launch_residual_norm(const NormParams &p, int dtype, int param_dtype, bool vec,
                                 cudaStream_t s);
cudaError_t launch_residual_norm_bwd(const NormBwdParams &p, int dtype, int param_dtype, bool vec,
                                     cudaStream_t s, int *launches);

}  // namespace scmp
