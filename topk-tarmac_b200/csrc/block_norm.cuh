// block_norm.cuh — parameters of the norms around a block (block_norm.cu).
#pragma once

#include "common.cuh"

namespace tarmac {

// episode and row stride of one [B, N, D] tensor, in elements
struct RowStrides {
  int64_t b, n;
};

struct NormParams {
  const void *x, *y, *gate;       // gate: or NULL (ones)
  const void *dh, *dz;            // backward: gradients of h and z, or NULL (zeros)
  void *h, *z;                    // forward, contiguous
  void *dx, *dy, *dgate;          // backward, contiguous
  RowStrides sx, sy, sg, sdh, sdz;
  const float *w_post, *w_pre, *scale;      // [D] or NULL (ones)
  float *dw_post, *dw_pre, *dscale;         // [D] or NULL
  float* work;                    // backward: [blocks][2][D] sums
  int B, N, D;
  float eps;
};

constexpr int NORM_MAX_D = 8192;

cudaError_t launch_residual_norm(const NormParams& p, bool bf16, cudaStream_t s);
cudaError_t launch_residual_norm_bwd(const NormParams& p, bool bf16, cudaStream_t s);
// floats of `work` that the backward call needs at most
int64_t residual_norm_bwd_work(int64_t rows, int D);

}  // namespace tarmac
