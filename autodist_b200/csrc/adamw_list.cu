// AdamW over a list of tensors in one launch, moments in fp32 or in 8 bits:
//
//   p *= 1 - lr wd;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p -= lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8 bits: every 256 elements of a tensor share a scale (the largest size over 448), m and the root of v are e4m3 values in it. The update
// itself uses the moments before they are rounded. A step moves v by a thousandth, which rounding to the nearest of values six per cent
// apart would undo every time, so values are rounded up or down at random with the probability of what is cut off, which keeps their
// mean. The random 16 bits are a hash of (seed, step, place), so a step can be repeated. A size that is not zero never becomes the
// value zero: a lost root would divide by eps alone.
//
// Measured (B200, fp32 parameters and gradients): 143 M parameters in 34 tensors, 8 bits 464 us (0.75 of the copy rate: 79 instructions a
// parameter, of which the memory would allow 88 with every issue slot taken), 32 bits 720 (0.85); 80 tensors of 4001 9.1 and 6.9. Steps that gave it: eight neighbours a lane 1278 -> 788 us, one hash for two of them and
// the rounding on exponents that coincide 634, 64 registers and the integer maximum of a warp 464.
#include "adamw_list.h"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "pdl.cuh"
#include "sm_count.h"

namespace adb200 {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int kThreads = 256;
constexpr int kChunk = 4096;                             // elements of a tensor that a thread block updates at a time
constexpr int kBlocks8 = 4, kBlocks32 = 4;               // on an SM
constexpr float kE4m3Max = 448.0f;
constexpr float kTiniest = 7.888609052210118e-31f;       // 2^-100: blocks below are held as zeros, their scale's inverse would overflow

// A launch copies its parameters: few tensors travel in a small table.
template <int MOST> struct Table {
  int count;
  int first[MOST + 1];                                   // chunks of the tensors in front
  AdamwTensor t[MOST];
};
static_assert(sizeof(Table<kAdamwMost>) + 256 <= 32764, "kernel parameters");

// 64 mixed bits of a counter, as the dropout decisions use them
constexpr uint64_t kGolden = 0x9E3779B97F4A7C15ull;
__device__ __forceinline__ uint64_t mixed(uint64_t x) {
  x ^= x >> 30; x *= 0xBF58476D1CE4E5B9ull;
  x ^= x >> 27; x *= 0x94D049BB133111EBull;
  return x ^ (x >> 31);
}

// two last bits off at most, of a step that is itself small beside the parameter
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The e4m3 code of a size (at most 448 and seven last bits), rounded up where the cut-off part and u = (bits16 + 1/2) / 65536 add up to one;
// `random`: 16 bits << 4 | 8. A code is a float's exponent and upper three bits of the fraction. Times 2^-120 the two types' exponents
// coincide, their subnormal numbers included (what is cut off there is below u's last bit), so that u is added below the fraction and
// what carries over is the rounding: 448 has no lower bits that could carry past the largest code. Nothing but zero becomes zero.
__device__ __forceinline__ uint32_t round_random(float size, uint32_t random) {
  uint32_t code = (__float_as_uint(__fmul_rz(size, 7.52316384526264e-37f)) + random) >> 20;
  if (size > 0.f) code = max(code, 1u);
  return code;
}

// Two e4m3 codes of a word's lower half
__device__ __forceinline__ float2 of_e4m3x2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  return __half22float2(__half2(h));
}

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
  s.key = mixed(r.seed + (uint64_t)t * kGolden);
  return s;
}
// Moments and parameter of one element; `root`: of the new second moment. The moments' roundings are spelled out, so that every kernel and
// the host's expressions round the same numbers to 8 bits: a last bit more or less decides now and then which of two values a moment becomes.
__device__ __forceinline__ void update(const Step& s, float& p, float g, float& m, float& v, float& root) {
  m = __fadd_rn(__fmul_rn(s.b1, m), __fmul_rn(s.c1, g));
  v = __fadd_rn(__fmul_rn(s.b2, v), __fmul_rn(s.c2, __fmul_rn(g, g)));
  root = __fsqrt_rn(v);
  p = fmaf(-s.rate * m, rcp_fast(fmaf(root, s.spread, s.eps)), p * s.decay);
}

// Eight neighbouring elements, of which `n` are there (8 or more: all, on 16 bytes).
__device__ __forceinline__ void load8(const float* p, int n, bool whole, float* v) {
  if (whole) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? p[j] : 0.f;
  }
}
__device__ __forceinline__ void load8(const bf16* p, int n, bool whole, float* v) {
  if (whole) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? __bfloat162float(p[j]) : 0.f;
  }
}
__device__ __forceinline__ void store8(float* p, int n, bool whole, const float* v) {
  if (whole) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) p[j] = v[j];
  }
}
__device__ __forceinline__ void store8(bf16* p, int n, bool whole, const float* v) {
  if (whole) {
    uint4 a;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&a);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    *reinterpret_cast<uint4*>(p) = a;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) p[j] = __float2bfloat16(v[j]);
  }
}

// A warp updates 256 elements at a time, a lane eight neighbours of them, so that the largest moments are found in registers and every byte
// moves once. Blocks walk along the list's chunks: what a step's elements share (two powers in double) is computed once for each.
template <typename P, typename G, bool BITS8, int MOST>
__global__ void __launch_bounds__(kThreads, 4) adamw_list_kernel(const __grid_constant__ Table<MOST> table, const AdamwMoments mo, const AdamwRule rule) {
  __shared__ Step shared;
  pdl_sync();
  if (threadIdx.x == 0) shared = step_of(rule, rule.step[0] + 1);
  __syncthreads();
  const Step s = shared;
  const int lane = threadIdx.x & 31, chunks = table.first[table.count];
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    int lo = 0, hi = table.count;              // the tensor whose chunk this is
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (table.first[mid] <= chunk) lo = mid; else hi = mid;
    }
    const AdamwTensor& t = table.t[lo];
    P* const params = static_cast<P*>(t.p);
    const G* const grads = static_cast<const G*>(t.g);
    const long long size = t.n, start = (long long)(chunk - table.first[lo]) * kChunk;
    const bool vectors = ((reinterpret_cast<uintptr_t>(params) | reinterpret_cast<uintptr_t>(grads)) & 15) == 0;
    for (int k = (threadIdx.x >> 5) * kAdamwBlock; k < kChunk && start + k < size; k += kThreads / 32 * kAdamwBlock) {
      const long long i = start + k + 8 * lane, q = t.place + i, block = (t.place + start + k) / kAdamwBlock;
      const int n = size - i > 8 ? 8 : (int)(size - i);  // of this lane's elements, can be none
      const bool whole = vectors && n == 8;
      float p[8], g[8], m[8], v[8], root[8];
      load8(params + i, n, whole, p);
      load8(grads + i, n, whole, g);
      if (BITS8) {                                       // moments are padded to whole blocks
        const uint2 mc = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(mo.m) + q)), rc = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(mo.r) + q));
        const float m_scale = mo.m_scale[block], r_scale = mo.r_scale[block];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 a = of_e4m3x2((j < 2 ? mc.x : mc.y) >> (16 * (j & 1)) & 0xFFFFu), b = of_e4m3x2((j < 2 ? rc.x : rc.y) >> (16 * (j & 1)) & 0xFFFFu);
          m[2 * j] = __fmul_rn(a.x, m_scale); m[2 * j + 1] = __fmul_rn(a.y, m_scale);
          v[2 * j] = __fmul_rn(b.x, r_scale); v[2 * j + 1] = __fmul_rn(b.y, r_scale);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], v[j]);
      } else {
        load8(static_cast<const float*>(mo.m) + q, 8, true, m);
        load8(static_cast<const float*>(mo.r) + q, 8, true, v);
      }
      float m_most = 0.f, r_most = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        update(s, p[j], g[j], m[j], v[j], root[j]);
        if (BITS8) {                                     // elements that are not there are zeros, as are their moments
          m_most = max_nan(m_most, fabsf(m[j]));
          r_most = max_nan(r_most, root[j]);
        }
      }
      store8(params + i, n, whole, p);
      if (BITS8) {
        // sizes compare as their bits do, NaN above infinity
        m_most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m_most)));
        r_most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(r_most)));
        const bool m_held = !(m_most < kTiniest), r_held = !(r_most < kTiniest);
        const float m_inv = m_held ? __fmul_rn(__frcp_rn(m_most), kE4m3Max) : 0.f, r_inv = r_held ? __fmul_rn(__frcp_rn(r_most), kE4m3Max) : 0.f;
        uint32_t mc[2] = {0u, 0u}, rc[2] = {0u, 0u};
        uint64_t counter = s.key + ((uint64_t)q >> 1) * kGolden;               // a hash for two neighbours
#pragma unroll
        for (int j = 0; j < 8; j += 2, counter += kGolden) {
          const uint64_t word = mixed(counter);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t bits = (uint32_t)(word >> (32 * h)), at = 8 * ((j + h) & 3);
            const float x = __fmul_rn(m[j + h], m_inv);
            const uint32_t code = round_random(fabsf(x), (bits << 4 & 0xFFFF0u) | 8u) | (__float_as_uint(x) >> 24 & 0x80u);
            mc[j >> 2] += code << at;
            rc[j >> 2] += round_random(__fmul_rn(root[j + h], r_inv), (bits >> 12 & 0xFFFF0u) | 8u) << at;
          }
        }
        // a block with a moment that is not finite is spoilt as a whole where its scale is NaN, else where the moment is not finite
        if (!(m_most < __int_as_float(0x7F800000)) || !(r_most < __int_as_float(0x7F800000))) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (isnan(m[j] * m_inv)) mc[j >> 2] |= 0x7Fu << (8 * (j & 3));
            if (isnan(root[j] * r_inv)) rc[j >> 2] |= 0x7Fu << (8 * (j & 3));
          }
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(mo.m) + q) = make_uint2(mc[0], mc[1]);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(mo.r) + q) = make_uint2(rc[0], rc[1]);
        if (lane == 0) {
          mo.m_scale[block] = m_held ? __fmul_rn(m_most, 1.0f / kE4m3Max) : 0.f;
          mo.r_scale[block] = r_held ? __fmul_rn(r_most, 1.0f / kE4m3Max) : 0.f;
        }
      } else {
        store8(static_cast<float*>(mo.m) + q, n, n == 8, m);
        store8(static_cast<float*>(mo.r) + q, n, n == 8, v);
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

template <typename P, typename G, int MOST>
cudaError_t step_of_list(const AdamwTensor* tensors, int count, const AdamwMoments& mo, const AdamwRule& rule, cudaStream_t st) {
  Table<MOST> table;
  table.count = count;
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    table.first[i] = (int)chunks;
    table.t[i] = tensors[i];
    chunks += (tensors[i].n + kChunk - 1) / kChunk;
    if (chunks > 0x7fffffffLL) return cudaErrorInvalidValue;
  }
  table.first[count] = (int)chunks;
  const long long most = (long long)sm_count() * (mo.m_scale != nullptr ? kBlocks8 : kBlocks32);
  return launch_pdl(mo.m_scale != nullptr ? adamw_list_kernel<P, G, true, MOST> : adamw_list_kernel<P, G, false, MOST>, dim3((unsigned)(chunks < most ? chunks : most)),
                    dim3(kThreads), 0, st, table, mo, rule);
}
template <typename P, typename G>
cudaError_t step_of_types(const AdamwTensor* tensors, int count, const AdamwMoments& mo, const AdamwRule& rule, cudaStream_t st) {
  return count <= 96 ? step_of_list<P, G, 96>(tensors, count, mo, rule, st) : step_of_list<P, G, kAdamwMost>(tensors, count, mo, rule, st);
}

}  // namespace

cudaError_t adamw_list_step(const AdamwTensor* tensors, int count, bool p_bf16, bool g_bf16, const AdamwMoments& mo, const AdamwRule& rule, cudaStream_t st) {
  if (count <= 0 || count > kAdamwMost) return cudaErrorInvalidValue;
  if (p_bf16) return g_bf16 ? step_of_types<bf16, bf16>(tensors, count, mo, rule, st) : step_of_types<bf16, float>(tensors, count, mo, rule, st);
  return g_bf16 ? step_of_types<float, bf16>(tensors, count, mo, rule, st) : step_of_types<float, float>(tensors, count, mo, rule, st);
}

}  // namespace adb200
