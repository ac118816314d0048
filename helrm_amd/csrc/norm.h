// norm.h -- launches of norm.hip.
#pragma once
#include "cleartext.h"

struct NormArgs {
  const void* x; long ldx;          // [rows][width], rows ldx elements apart
  const void* weight; const void* bias;
  void* y; long ldy;                // forward: the output; backward: its gradient
  float* mean; float* rstd;         // [rows]; the forward's may be null
  void* dx; long lddx;              // backward
  void* dweight; void* dbias;
  void* workspace;
  long rows; int width, dtype, param_dtype;
  float eps;
};
void norm_forward_launch(const NormArgs& a, hipStream_t st);
size_t norm_backward_workspace(long rows, int width);
void norm_backward_launch(const NormArgs& a, hipStream_t st);
