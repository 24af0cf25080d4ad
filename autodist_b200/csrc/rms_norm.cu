// Root-mean-square norm over rows, with the residual's addition in front of it, its gradient, and rows in 8 bits with a scale each.
//
//   s = x + res, rounded to the stream's type: what leaves is what is normed
//   y = s * rstd * w,  rstd = 1 / sqrt(mean(s^2) + eps)
//   8 bits: scale = max |y| / 448, code = e4m3(y / scale)
//   dx = ds + rstd * (g - n * mean(g n)),  dw = sum over rows of dy * n,  with g = dy * w, n = s * rstd
//
// Sums are fp32. Memory-bound: a few operations for each element that is read and written once.
#include "rms_norm.h"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "pdl.cuh"
#include "sm_count.h"

namespace adb200 {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int kThreads = 256;
constexpr float kE4m3Max = 448.0f;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16(v); }

// The larger of two numbers; NaN when one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return max_nan(a, b); } };

template <class Op>
__device__ __forceinline__ float block_all(float v, float* shared, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();                                    // the last use of `shared` is over
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < kThreads / 32; ++w) v = op(v, shared[w]);
  return v;
}

// A block per row; QUANT: rows leave in 8 bits. The row is read again where it is needed again.
template <typename T, typename W, bool QUANT>
__global__ void __launch_bounds__(kThreads) norm_kernel(const NormRows p, T* __restrict__ y, uint8_t* __restrict__ codes, long long codes_ld,
                                                        float* __restrict__ scales) {
  pdl_sync();
  __shared__ float shared[kThreads / 32];
  const W* w = static_cast<const W*>(p.weight);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
    const T* res = p.res != nullptr ? static_cast<const T*>(p.res) + row * p.res_ld : nullptr;
    T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + row * p.width : nullptr;
    auto element = [&](int c) { return res != nullptr ? to_f(from_f<T>(to_f(x[c]) + to_f(res[c]))) : to_f(x[c]); };
    float rstd = 1.0f;
    if (w != nullptr) {
      float q = 0.f;
      for (int c = threadIdx.x; c < p.width; c += kThreads) {
        const float v = element(c);
        q += v * v;
      }
      rstd = rsqrtf(block_all(q, shared, Add()) / p.width + p.eps);
    }
    auto normed = [&](int c) { return w != nullptr ? element(c) * rstd * to_f(w[c]) : element(c); };
    float inv = 0.f;
    if (QUANT) {
      float most = 0.f;
      for (int c = threadIdx.x; c < p.width; c += kThreads) most = max_nan(most, fabsf(normed(c)));
      most = block_all(most, shared, Max());
      const float scale = most / kE4m3Max;
      if (threadIdx.x == 0) scales[row] = scale;
      inv = scale == 0.f ? 0.f : 1.0f / scale;
    }
    for (int c = threadIdx.x; c < p.width; c += kThreads) {
      if (sum != nullptr) sum[c] = from_f<T>(element(c));
      if (QUANT)
        codes[row * codes_ld + c] = __nv_cvt_float_to_fp8(normed(c) * inv, __NV_SATFINITE, __NV_E4M3);
      else
        y[row * p.width + c] = from_f<T>(normed(c));
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) norm_dx_kernel(const NormGrad p, float* __restrict__ rstds) {
  pdl_sync();
  __shared__ float shared[kThreads / 32];
  const W* w = static_cast<const W*>(p.weight);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* s = static_cast<const T*>(p.s) + row * p.s_ld;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dy_ld;
    const T* ds = p.ds != nullptr ? static_cast<const T*>(p.ds) + row * p.ds_ld : nullptr;
    float q = 0.f, d = 0.f;
    for (int c = threadIdx.x; c < p.width; c += kThreads) {
      const float v = to_f(s[c]);
      q += v * v;
      d += v * to_f(dy[c]) * to_f(w[c]);
    }
    q = block_all(q, shared, Add());
    d = block_all(d, shared, Add());
    const float rstd = rsqrtf(q / p.width + p.eps), along = d * rstd / p.width;
    if (threadIdx.x == 0) rstds[row] = rstd;
    for (int c = threadIdx.x; c < p.width; c += kThreads) {
      float v = rstd * (to_f(dy[c]) * to_f(w[c]) - to_f(s[c]) * rstd * along);
      if (ds != nullptr) v += to_f(ds[c]);
      static_cast<T*>(p.dx)[row * p.width + c] = from_f<T>(v);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) norm_dw_kernel(const NormGrad p, const float* __restrict__ rstds, float* __restrict__ part, int parts) {
  pdl_sync();
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= p.width) return;
  float sum = 0.f;
  for (long long row = blockIdx.y; row < p.rows; row += parts)
    sum += to_f(static_cast<const T*>(p.dy)[row * p.dy_ld + c]) * to_f(static_cast<const T*>(p.s)[row * p.s_ld + c]) * rstds[row];
  part[(long long)blockIdx.y * p.width + c] = sum;
}

template <typename W>
__global__ void __launch_bounds__(kThreads) norm_dw_sum_kernel(const float* __restrict__ part, W* __restrict__ dw, int parts, int width) {
  pdl_sync();
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= width) return;
  float sum = 0.f;
  for (int k = 0; k < parts; ++k) sum += part[(long long)k * width + c];
  dw[c] = from_f<W>(sum);
}

template <typename T, typename W, bool QUANT>
cudaError_t forward(const NormRows& p, void* y, void* codes, long long codes_ld, float* scales, cudaStream_t st) {
  if (p.rows <= 0) return cudaSuccess;
  const long long most = 8LL * sm_count();
  return launch_pdl(norm_kernel<T, W, QUANT>, dim3((unsigned)(p.rows < most ? p.rows : most)), dim3(kThreads), 0, st, p, static_cast<T*>(y),
                    static_cast<uint8_t*>(codes), codes_ld, scales);
}
template <bool QUANT>
cudaError_t forward_of(const NormRows& p, void* y, void* codes, long long codes_ld, float* scales, cudaStream_t st) {
  if (!p.bf16) return p.weight_bf16 ? cudaErrorInvalidValue : forward<float, float, QUANT>(p, y, codes, codes_ld, scales, st);
  return p.weight_bf16 ? forward<bf16, bf16, QUANT>(p, y, codes, codes_ld, scales, st) : forward<bf16, float, QUANT>(p, y, codes, codes_ld, scales, st);
}

constexpr int kParts = 64;

template <typename T, typename W>
cudaError_t backward(const NormGrad& p, cudaStream_t st) {
  const int parts = rms_norm_bwd_parts(p.rows, p.width) - (int)((p.rows + p.width - 1) / p.width);
  float* rstds = p.part + (long long)parts * p.width;
  const unsigned cols = (p.width + kThreads - 1) / kThreads;
  cudaError_t e = cudaSuccess;
  if (p.rows > 0) {
    const long long most = 8LL * sm_count();
    e = launch_pdl(norm_dx_kernel<T, W>, dim3((unsigned)(p.rows < most ? p.rows : most)), dim3(kThreads), 0, st, p, rstds);
    if (e == cudaSuccess) e = launch_pdl(norm_dw_kernel<T>, dim3(cols, parts), dim3(kThreads), 0, st, p, rstds, p.part, parts);
  }
  if (e == cudaSuccess) e = launch_pdl(norm_dw_sum_kernel<W>, dim3(cols), dim3(kThreads), 0, st, p.part, static_cast<W*>(p.dw), p.rows > 0 ? parts : 0, p.width);
  return e;
}

}  // namespace

cudaError_t rms_norm_fwd(const NormRows& p, void* y, cudaStream_t st) { return forward_of<false>(p, y, nullptr, 0, nullptr, st); }
cudaError_t rms_norm_8bit(const NormRows& p, void* codes, long long codes_ld, float* scales, cudaStream_t st) {
  return forward_of<true>(p, nullptr, codes, codes_ld, scales, st);
}
int rms_norm_bwd_parts(long long rows, int width) { return kParts + (int)((rows + width - 1) / width); }      // the rows' rstd behind the sums
cudaError_t rms_norm_bwd(const NormGrad& p, cudaStream_t st) {
  if (!p.bf16) return p.weight_bf16 ? cudaErrorInvalidValue : backward<float, float>(p, st);
  return p.weight_bf16 ? backward<bf16, bf16>(p, st) : backward<bf16, float>(p, st);
}

}  // namespace adb200
