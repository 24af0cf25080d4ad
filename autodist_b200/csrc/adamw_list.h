// Host-side interface of the AdamW step over a list of tensors (see adamw_list.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace adb200 {

constexpr int kAdamwBlock = 256;           // elements of a tensor that share a scale of the 8-bit moments; every tensor's moments start on one
constexpr int kAdamwMost = 640;            // tensors of a launch: their table travels as a kernel parameter

struct AdamwTensor {
  void* p;
  const void* g;
  long long n;
  long long place;                         // where its moments start, a multiple of kAdamwBlock
};
struct AdamwRule {
  double b1, b2, eps, wd;
  const float* lr_at;                      // device scalar, or nullptr: `lr`
  double lr;
  unsigned long long seed;
  long long* step;                         // [0]: steps taken, [1]: blocks of the running launch that are done (0 between calls)
  int advance;                             // whether this launch is the step's last, which counts it
};
struct AdamwMoments {
  void *m, *r;                             // fp32 moments, or e4m3 values of the first moment and of the root of the second
  float *m_scale, *r_scale;                // per block of kAdamwBlock; nullptr: fp32 moments
};
// `tensors`: at most kAdamwMost, none of them empty
cudaError_t adamw_list_step(const AdamwTensor* tensors, int count, bool p_bf16, bool g_bf16, const AdamwMoments& moments, const AdamwRule& rule, cudaStream_t st);

}  // namespace adb200
