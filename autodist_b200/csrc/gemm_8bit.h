// Host-side interface of the product of rows in 8 bits (see gemm_8bit.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace adb200 {

// y[m, n] = scales[m] * weight_scales[n] * sum_k codes[m, k] weight_codes[n, k] + bias[n], e4m3 codes, bf16 result. `*_ld`: bytes between rows, a
// multiple of 16; codes, scales and bias start on 16-byte boundaries.
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
// `bn`: rows of `codes` in a tile (16, 32, 64, 128; 512: the kernel on SM pairs), `split`: how many CTAs share a contraction (1 to 8); 0: chosen
cudaError_t gemm_8bit(const Gemm8Args& a, int bn, int split, cudaStream_t st);

}  // namespace adb200
