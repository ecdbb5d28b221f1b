// Launch interface of the layer norm kernels.
#pragma once

#include <cuda_runtime.h>

namespace prism {

struct NormArgs {
  const void* x;          // forward: x; backward: what was normalised (x, or the sum)
  const void* residual;   // forward: added to x, or null
  const void *weight, *bias;   // [cols], fp32 (w_f32) or of the rows' type; bias may be null
  void *y, *sum;          // forward outputs, contiguous; sum only with residual
  float *mean, *rstd;     // [rows]; forward: may be null
  const void *dy, *dsum;  // backward; dsum may be null
  void* dx;               // contiguous
  void *dw, *db;          // [cols], as weight; db may be null
  float* partial;         // backward scratch [ctas][2][cols]
  int ctas;
  long long rows;
  int cols;
  long long ldx, ldr, lddy, ldds;
  float eps;
  int dtype;
  bool w_f32;
  cudaStream_t stream;
};

int norm_max_cols();
int norm_bwd_ctas(long long rows, int cols, int num_sms);
int launch_norm_fwd(const NormArgs& a);
int launch_norm_bwd(const NormArgs& a);

}  // namespace prism
