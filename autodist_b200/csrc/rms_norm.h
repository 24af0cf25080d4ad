// Host-side interface of the root-mean-square norm and of the rows in 8 bits (see rms_norm.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace adb200 {

// Rows of `width` elements; `*_ld`: elements from one row to the next. `bf16`: the stream's type (else fp32); `weight_bf16`: the weight's.
struct NormRows {
  const void* x; long long x_ld;
  const void* res; long long res_ld;        // nullptr: no residual
  const void* weight;
  void* sum;                                // [rows, width]: x + res, nullptr without a residual
  long long rows; int width; float eps;
  bool bf16, weight_bf16;
};
// y: [rows, width] of the stream's type
cudaError_t rms_norm_fwd(const NormRows& p, void* y, cudaStream_t st);
// codes: [rows, codes_ld] e4m3, scales: [rows]. Without a weight (nullptr) the rows themselves are rounded.
cudaError_t rms_norm_8bit(const NormRows& p, void* codes, long long codes_ld, float* scales, cudaStream_t st);

struct NormGrad {
  const void* dy; long long dy_ld;
  const void* ds; long long ds_ld;          // gradient that reaches the sum by itself; nullptr: none
  const void* s; long long s_ld;            // what was normed
  const void* weight;
  void* dx;                                 // [rows, width]
  float* part;                              // rms_norm_bwd_floats(p)
  void* dw;                                 // [width] of the weight's type
  long long rows; int width; float eps;
  bool bf16, weight_bf16;
};
// Floats of scratch (all but `part` and `dw` have to be set); launched: how many kernels it took.
long long rms_norm_bwd_floats(const NormGrad& p);
cudaError_t rms_norm_bwd(const NormGrad& p, int* launched, cudaStream_t st);

}  // namespace adb200
