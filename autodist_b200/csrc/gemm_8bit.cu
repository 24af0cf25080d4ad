// Product of rows in 8 bits with a scale each: y = (codes . weight_codes^T) * scales * weight_scales + bias, sums in fp32, bf16 result.
#include "gemm_8bit.h"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "pdl.cuh"

namespace adb200 {
namespace {

constexpr int kTile = 16;

__device__ __forceinline__ float of_e4m3(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }

// A 16 x 16 tile of the result per block, a value per thread.
__global__ void __launch_bounds__(kTile * kTile) gemm8_kernel(const Gemm8Args a) {
  pdl_sync();
  __shared__ float sx[kTile][kTile + 1], sw[kTile][kTile + 1];
  const int tiles_n = (a.N + kTile - 1) / kTile;
  const int m0 = blockIdx.x / tiles_n * kTile, n0 = blockIdx.x % tiles_n * kTile;
  const int tx = threadIdx.x % kTile, ty = threadIdx.x / kTile;
  float sum = 0.f;
  for (int k0 = 0; k0 < a.K; k0 += kTile) {
    const int k = k0 + tx;
    sx[ty][tx] = m0 + ty < a.M && k < a.K ? of_e4m3(a.codes[(long long)(m0 + ty) * a.codes_ld + k]) : 0.f;
    sw[ty][tx] = n0 + ty < a.N && k < a.K ? of_e4m3(a.weight_codes[(long long)(n0 + ty) * a.weight_ld + k]) : 0.f;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kTile; ++j) sum += sx[ty][j] * sw[tx][j];
    __syncthreads();
  }
  const int m = m0 + ty, n = n0 + tx;
  if (m < a.M && n < a.N) {
    const float v = sum * (a.scales[m] * a.weight_scales[n]) + (a.bias != nullptr ? a.bias[n] : 0.f);
    static_cast<__nv_bfloat16*>(a.y)[(long long)m * a.N + n] = __float2bfloat16(v);
  }
}

}  // namespace

cudaError_t gemm_8bit(const Gemm8Args& a, cudaStream_t st) {
  if (a.M <= 0 || a.N <= 0) return cudaSuccess;
  const long long tiles = (long long)((a.M + kTile - 1) / kTile) * ((a.N + kTile - 1) / kTile);
  if (tiles > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch_pdl(gemm8_kernel, dim3((unsigned)tiles), dim3(kTile * kTile), 0, st, a);
}

}  // namespace adb200
