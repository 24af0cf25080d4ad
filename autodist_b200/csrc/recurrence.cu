// Gated linear recurrence over time, channel by channel:
//
//   h_t = f_t h_{t-1} + u_t x_t,   f = sigmoid(forget + bias),   u = sigmoid(input), or 1 - f without an input gate
//
// and f_t counts as 0 in front of h_{t-1} where `reset` says that the state is forgotten. Backward:
//
//   dh_t = dy_t + f_{t+1} dh_{t+1},   dx = dh u,   dforget = dh (h_{t-1} [- x]) f (1 - f),   dinput = dh x u (1 - u)
//
// The states are not stored: the forward pass keeps them in fp32 in front of every tile of kScanTile steps, and the backward pass
// computes those in between again. States, gates and sums are fp32.
#include "recurrence.h"

#include <cuda_bf16.h>

#include "pdl.cuh"
#include "sm_count.h"

namespace adb200 {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int kThreads = 128;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16(v); }

// sigmoid(v) and 1 - sigmoid(v), neither of them by subtraction
__device__ __forceinline__ float2 both_sides(float v) {
  const float t = expf(-fabsf(v)), r = 1.0f / (1.0f + t);
  return v >= 0.f ? make_float2(r, t * r) : make_float2(t * r, r);
}

template <typename T> __device__ __forceinline__ const T* at(const ScanView& v, int b, int t) { return static_cast<const T*>(v.p) + b * v.batch + t * v.step; }

// A thread per channel walks through time.
template <typename T, bool GATE>
__global__ void __launch_bounds__(kThreads) scan_fwd_kernel(const ScanArgs a, T* __restrict__ y, float* __restrict__ last, float* __restrict__ kept) {
  pdl_sync();
  const int across = (a.channels + kThreads - 1) / kThreads;
  const int c = blockIdx.x % across * kThreads + threadIdx.x, b = blockIdx.x / across;
  if (c >= a.channels) return;
  const int tiles = (a.steps + kScanTile - 1) / kScanTile;
  float h = a.state != nullptr ? a.state[(long long)b * a.channels + c] : 0.f;
  for (int t = 0; t < a.steps; ++t) {
    if (kept != nullptr && t % kScanTile == 0) kept[((long long)b * tiles + t / kScanTile) * a.channels + c] = h;
    const float2 f = both_sides(to_f(at<T>(a.forget, b, t)[c]) + a.forget_bias);
    const float u = GATE ? both_sides(to_f(at<T>(a.input, b, t)[c])).x : f.y;
    const float v = u * to_f(at<T>(a.x, b, t)[c]);
    h = a.reset != nullptr && a.reset[b * a.reset_batch + t * a.reset_step] ? v : f.x * h + v;
    y[((long long)b * a.steps + t) * a.channels + c] = from_f<T>(h);
  }
  last[(long long)b * a.channels + c] = h;
}

template <typename T, bool GATE>
__global__ void __launch_bounds__(kThreads) scan_bwd_kernel(const ScanArgs a, const ScanGrads g) {
  pdl_sync();
  const int across = (a.channels + kThreads - 1) / kThreads;
  const int c = blockIdx.x % across * kThreads + threadIdx.x, b = blockIdx.x / across;
  if (c >= a.channels) return;
  const int tiles = (a.steps + kScanTile - 1) / kScanTile;
  float carry = g.dlast != nullptr ? g.dlast[(long long)b * a.channels + c] : 0.f;       // f_{t+1} dh_{t+1}
  for (int k = tiles - 1; k >= 0; --k) {
    const int t0 = k * kScanTile, n = min(kScanTile, a.steps - t0);
    float before[kScanTile];
    float h = g.kept[((long long)b * tiles + k) * a.channels + c];
    for (int i = 0; i < n; ++i) {
      const int t = t0 + i;
      const bool cut = a.reset != nullptr && a.reset[b * a.reset_batch + t * a.reset_step];
      before[i] = cut ? 0.f : h;
      const float2 f = both_sides(to_f(at<T>(a.forget, b, t)[c]) + a.forget_bias);
      const float u = GATE ? both_sides(to_f(at<T>(a.input, b, t)[c])).x : f.y;
      const float v = u * to_f(at<T>(a.x, b, t)[c]);
      h = cut ? v : f.x * h + v;
    }
    for (int i = n - 1; i >= 0; --i) {
      const int t = t0 + i;
      const bool cut = a.reset != nullptr && a.reset[b * a.reset_batch + t * a.reset_step];
      const float dh = carry + (g.dy.p != nullptr ? to_f(at<T>(g.dy, b, t)[c]) : 0.f);
      const float2 f = both_sides(to_f(at<T>(a.forget, b, t)[c]) + a.forget_bias);
      const float2 u = GATE ? both_sides(to_f(at<T>(a.input, b, t)[c])) : make_float2(f.y, f.x);
      const float x = to_f(at<T>(a.x, b, t)[c]);
      const long long out = ((long long)b * a.steps + t) * a.channels + c;
      static_cast<T*>(g.dx)[out] = from_f<T>(dh * u.x);
      static_cast<T*>(g.dforget)[out] = from_f<T>(dh * (GATE ? before[i] : before[i] - x) * f.x * f.y);
      if (GATE) static_cast<T*>(g.dinput)[out] = from_f<T>(dh * x * u.x * u.y);
      carry = cut ? 0.f : f.x * dh;
    }
  }
  g.dstate[(long long)b * a.channels + c] = carry;
}

}  // namespace

cudaError_t gated_scan_fwd(const ScanArgs& a, void* y, float* last, float* kept, cudaStream_t st) {
  if (a.batch <= 0 || a.channels <= 0) return cudaSuccess;
  const dim3 grid((a.channels + kThreads - 1) / kThreads * a.batch);
  const bool gate = a.input.p != nullptr;
  if (a.bf16) return launch_pdl(gate ? scan_fwd_kernel<bf16, true> : scan_fwd_kernel<bf16, false>, grid, dim3(kThreads), 0, st, a, static_cast<bf16*>(y), last, kept);
  return launch_pdl(gate ? scan_fwd_kernel<float, true> : scan_fwd_kernel<float, false>, grid, dim3(kThreads), 0, st, a, static_cast<float*>(y), last, kept);
}
cudaError_t gated_scan_bwd(const ScanArgs& a, const ScanGrads& g, cudaStream_t st) {
  if (a.batch <= 0 || a.channels <= 0) return cudaSuccess;
  const dim3 grid((a.channels + kThreads - 1) / kThreads * a.batch);
  const bool gate = a.input.p != nullptr;
  if (a.bf16) return launch_pdl(gate ? scan_bwd_kernel<bf16, true> : scan_bwd_kernel<bf16, false>, grid, dim3(kThreads), 0, st, a, g);
  return launch_pdl(gate ? scan_bwd_kernel<float, true> : scan_bwd_kernel<float, false>, grid, dim3(kThreads), 0, st, a, g);
}

}  // namespace adb200
