// Host-side interface of the gated linear recurrence (see recurrence.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace adb200 {

// [batch, steps, channels] views with unit stride along channels; strides in elements.
struct ScanView { const void* p; long long batch, step; };
struct ScanArgs {
  ScanView x, forget, input;               // input.p == nullptr: the input is weighted by 1 - forget
  const float* state;                      // [batch, channels]; nullptr: zeros
  const uint8_t* reset; long long reset_batch, reset_step;      // [batch, steps]; nullptr: none
  int batch, steps, channels;
  float forget_bias;
  bool bf16;                               // else fp32
};
// Steps between the states that the forward pass keeps for the backward pass; goes by the sizes alone.
int gated_scan_tile(const ScanArgs& a);
// y: [batch, steps, channels], last: [batch, channels]; kept (nullptr: not wanted): [batch, ceil(steps / gated_scan_tile), channels], the states
// in front of each tile
// runs: gated_scan_runs(a) floats of scratch, for either pass; launched: how many kernels it took
long long gated_scan_runs(const ScanArgs& a);
cudaError_t gated_scan_fwd(const ScanArgs& a, void* y, float* last, float* kept, float* runs, int* launched, cudaStream_t st);

struct ScanGrads {
  ScanView dy;                             // p == nullptr: zeros
  const float* dlast;                      // nullptr: zeros
  const float* kept;
  void *dx, *dforget, *dinput;             // [batch, steps, channels]; dinput only with an input gate
  float* dstate;                           // [batch, channels]
};
cudaError_t gated_scan_bwd(const ScanArgs& a, const ScanGrads& g, float* runs, int* launched, cudaStream_t st);

}  // namespace adb200
