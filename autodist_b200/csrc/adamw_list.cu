// AdamW over a list of tensors in one launch, moments in fp32 or in 8 bits:
//
//   p *= 1 - lr wd;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p -= lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8 bits: every 256 elements of a tensor share a scale (the largest size over 448), m and the root of v are e4m3 values in it. The update
// itself uses the moments before they are rounded. A step moves v by a thousandth, which rounding to the nearest of values six per cent
// apart would undo every time, so values are rounded up or down at random with the probability of what is cut off, which keeps their
// mean. The random 16 bits are a hash of (seed, step, place), so a step can be repeated. A size that is not zero never becomes the
// value zero: a lost root would divide by eps alone.
#include "adamw_list.h"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "pdl.cuh"

namespace adb200 {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int kThreads = 256;
constexpr float kE4m3Max = 448.0f;
constexpr float kTiniest = 7.888609052210118e-31f;        // 2^-100: blocks below are held as zeros, their scale's inverse would overflow
static_assert(sizeof(AdamwTable) + 256 <= 32764, "kernel parameters");

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16* p, float v) { *p = __float2bfloat16(v); }

// 64 mixed bits of a counter, as the dropout decisions use them
__device__ __forceinline__ uint64_t mixed(uint64_t seed, uint64_t i) {
  uint64_t x = seed + i * 0x9E3779B97F4A7C15ull;
  x ^= x >> 30; x *= 0xBF58476D1CE4E5B9ull;
  x ^= x >> 27; x *= 0x94D049BB133111EBull;
  return x ^ (x >> 31);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The e4m3 value at |v| <= 448 (and a rounding), rounded up where the cut-off part and the random 16 bits add up to one.
__device__ __forceinline__ uint8_t round_random(float v, uint32_t bits16) {
  const float size = fabsf(v);
  const uint32_t binade = __float_as_uint(fmaxf(size, 0.015625f)) & 0x7F800000u;       // the power of two below, 2^-6 for the smallest
  const float ulp = __uint_as_float(binade - (3u << 23)), inv = __uint_as_float((254u << 23) - (binade - (3u << 23)));
  const float u = ((float)bits16 + 0.5f) * (1.0f / 65536.0f);
  float q = floorf(__fadd_rn(__fmul_rn(size, inv), u)) * ulp;
  if (q > kE4m3Max) q = kE4m3Max;
  if (q == 0.f && size > 0.f) q = 0.001953125f;
  return __nv_cvt_float_to_fp8(copysignf(q, v), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float of_e4m3(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }

struct Step {
  float decay, rate, spread, b1, c1, b2, c2, eps;
  uint64_t key;
};
// What all elements of a step share. `t`: this step's number, from 1.
__device__ Step step_of(const AdamwRule& r, long long t) {
  const double lr = r.lr_at != nullptr ? (double)*r.lr_at : r.lr;
  Step s;
  s.decay = (float)(1.0 - lr * r.wd);
  s.rate = (float)(lr / (1.0 - pow(r.b1, (double)t)));
  s.spread = (float)(1.0 / sqrt(1.0 - pow(r.b2, (double)t)));
  s.b1 = (float)r.b1; s.c1 = (float)(1.0 - r.b1); s.b2 = (float)r.b2; s.c2 = (float)(1.0 - r.b2); s.eps = (float)r.eps;
  s.key = mixed(r.seed, (uint64_t)t);
  return s;
}
// Moments and parameter of one element; `root`: of the new second moment. The moments' roundings are spelled out, so that every kernel and
// the host's expressions round the same numbers to 8 bits: a last bit more or less decides now and then which of two values a moment becomes.
__device__ __forceinline__ void update(const Step& s, float& p, float g, float& m, float& v, float& root) {
  m = __fadd_rn(__fmul_rn(s.b1, m), __fmul_rn(s.c1, g));
  v = __fadd_rn(__fmul_rn(s.b2, v), __fmul_rn(s.c2, __fmul_rn(g, g)));
  root = __fsqrt_rn(v);
  p = p * s.decay - s.rate * (m / (root * s.spread + s.eps));
}

// A thread block per chunk of a tensor; a warp's blocks of 256 elements one after the other.
template <typename P, typename G, bool BITS8>
__global__ void __launch_bounds__(kThreads) adamw_list_kernel(const __grid_constant__ AdamwTable table, const AdamwMoments mo, const AdamwRule rule) {
  pdl_sync();
  __shared__ Step shared;
  if (threadIdx.x == 0) shared = step_of(rule, rule.step[0] + 1);
  __syncthreads();
  const Step s = shared;
  const int chunk = blockIdx.x;
  int lo = 0, hi = table.count;              // the tensor whose chunk this is
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (table.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  const AdamwTensor t = table.t[lo];
  const long long start = (long long)(chunk - table.first[lo]) * kAdamwChunk;
  const int lane = threadIdx.x & 31;
  for (int k = (threadIdx.x >> 5) * kAdamwBlock; k < kAdamwChunk && start + k < t.n; k += kThreads / 32 * kAdamwBlock) {
    const long long place = t.place + start + k;
    float m[8], root[8];
    float m_most = 0.f, r_most = 0.f;
    const float m_scale = BITS8 ? mo.m_scale[place / kAdamwBlock] : 0.f, r_scale = BITS8 ? mo.r_scale[place / kAdamwBlock] : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long i = start + k + 32 * j + lane;
      const long long q = place + 32 * j + lane;
      m[j] = root[j] = 0.f;
      if (i < t.n) {
        float v;
        if (BITS8) {
          m[j] = __fmul_rn(of_e4m3(static_cast<const uint8_t*>(mo.m)[q]), m_scale);
          v = __fmul_rn(of_e4m3(static_cast<const uint8_t*>(mo.r)[q]), r_scale);
          v = __fmul_rn(v, v);
        } else {
          m[j] = static_cast<const float*>(mo.m)[q];
          v = static_cast<const float*>(mo.r)[q];
        }
        P* pp = static_cast<P*>(t.p) + i;
        float p = to_f(*pp);
        update(s, p, to_f(static_cast<const G*>(t.g)[i]), m[j], v, root[j]);
        put(pp, p);
        if (!BITS8) {
          static_cast<float*>(mo.m)[q] = m[j];
          static_cast<float*>(mo.r)[q] = v;
        }
        m_most = max_nan(m_most, fabsf(m[j]));
        r_most = max_nan(r_most, root[j]);
      }
    }
    if (BITS8) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        m_most = max_nan(m_most, __shfl_xor_sync(0xffffffffu, m_most, o));
        r_most = max_nan(r_most, __shfl_xor_sync(0xffffffffu, r_most, o));
      }
      const bool m_held = !(m_most < kTiniest), r_held = !(r_most < kTiniest);
      const float m_inv = m_held ? __fmul_rn(__frcp_rn(m_most), kE4m3Max) : 0.f, r_inv = r_held ? __fmul_rn(__frcp_rn(r_most), kE4m3Max) : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const long long i = start + k + 32 * j + lane;
        const long long q = place + 32 * j + lane;
        if (i < t.n) {
          const uint64_t word = mixed(s.key, (uint64_t)q >> 1);
          const uint32_t bits = (uint32_t)(word >> ((q & 1) * 32));
          static_cast<uint8_t*>(mo.m)[q] = round_random(__fmul_rn(m[j], m_inv), bits & 0xFFFFu);
          static_cast<uint8_t*>(mo.r)[q] = round_random(__fmul_rn(root[j], r_inv), bits >> 16);
        }
      }
      if (lane == 0) {
        mo.m_scale[place / kAdamwBlock] = m_held ? __fmul_rn(m_most, 1.0f / kE4m3Max) : 0.f;
        mo.r_scale[place / kAdamwBlock] = r_held ? __fmul_rn(r_most, 1.0f / kE4m3Max) : 0.f;
      }
    }
  }
  // The block that finishes last counts the step: all others have read the count by then.
  if (rule.advance && threadIdx.x == 0) {
    const unsigned long long done = atomicAdd(reinterpret_cast<unsigned long long*>(rule.step + 1), 1ull);
    if (done == gridDim.x - 1) {
      rule.step[1] = 0;
      rule.step[0] += 1;
    }
  }
}

template <typename P, typename G>
cudaError_t step_of_types(const AdamwTable& table, const AdamwMoments& mo, const AdamwRule& rule, cudaStream_t st) {
  const dim3 grid((unsigned)table.first[table.count]);
  return launch_pdl(mo.m_scale != nullptr ? adamw_list_kernel<P, G, true> : adamw_list_kernel<P, G, false>, grid, dim3(kThreads), 0, st, table, mo, rule);
}

}  // namespace

cudaError_t adamw_list_step(const AdamwTable& table, bool p_bf16, bool g_bf16, const AdamwMoments& mo, const AdamwRule& rule, cudaStream_t st) {
  if (table.count <= 0 || table.first[table.count] <= 0) return cudaErrorInvalidValue;
  if (p_bf16) return g_bf16 ? step_of_types<bf16, bf16>(table, mo, rule, st) : step_of_types<bf16, float>(table, mo, rule, st);
  return g_bf16 ? step_of_types<float, bf16>(table, mo, rule, st) : step_of_types<float, float>(table, mo, rule, st);
}

}  // namespace adb200
