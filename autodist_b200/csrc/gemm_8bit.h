// Host-side interface of the product of rows in 8 bits (see gemm_8bit.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace adb200 {

// y[m, n] = scales[m] * weight_scales[n] * sum_k codes[m, k] weight_codes[n, k] + bias[n], e4m3 codes, bf16 result. `*_ld`: elements (bytes)
// between rows, multiples of 16, bases on 16 bytes.
struct Gemm8Args {
  const uint8_t* codes; long long codes_ld;
  const float* scales;
  const uint8_t* weight_codes; long long weight_ld;
  const float* weight_scales;
  const float* bias;                       // nullptr: none
  void* y;                                 // bf16 [M, N]
  int M, N, K;
  int* error;                              // where a kernel that gave up waiting writes its code
};
cudaError_t gemm_8bit(const Gemm8Args& a, cudaStream_t st);

}  // namespace adb200
