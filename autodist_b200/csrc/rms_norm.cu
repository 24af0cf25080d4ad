// Root-mean-square norm over rows, with the residual's addition in front of it, its gradient, and rows in 8 bits with a scale each.
//
//   s = x + res, rounded to the stream's type: what leaves is what is normed
//   y = s * rstd * w,  rstd = 1 / sqrt(mean(s^2) + eps)
//   8 bits: scale = max |y| / 448, code = e4m3(y / scale)
//   dx = ds + rstd * (g - n * mean(g n)),  dw = sum over rows of dy * n,  with g = dy * w, n = s * rstd
//
// Sums are fp32. Memory-bound: a few operations for each element that is read and written once. A row stays in the registers of the 32 to
// 512 threads that share it (16 bytes a piece), so that it is read once; thread groups walk along the rows with the weight, and backward
// the weight's gradient, of their columns in registers too. Rows wider than that are read again for every sum.
//
// Measured (B200, replayed back to back; shares of the copy rate): 16384 x 4096 in bf16 with a residual, forward 101 us (0.81), in 8 bits 78
// (0.92), backward 98 (0.83); 32768 x 1024 in fp32 86, 74, 86 (0.95, 0.90, 0.95); 12289 x 1001 in fp32 without a residual 22 and 35; 8 x 2048
// 2.4 and 4.7, a launch each. What held it back before was the wait for a row behind every row's sums: with the next row's pieces in
// registers 151 us backward where rows ahead in shared memory take 98; with the largest size in an exchange of its own 108 us in 8 bits
// where one exchange for both takes 97, and rows ahead 78. What it has not solved are the widest
// odd rows in bf16: 4096 x 8191 takes 64 us forward and 119 backward where 8185 columns take 34 and 69, since its 1025 pieces need four a
// thread.
#include "rms_norm.h"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <mutex>
#include <set>

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

// ------------------------------------------------------------------------------------------------ rows in registers
// VEC neighbouring elements as they lie in memory.
template <typename T, int VEC> struct Piece;
template <> struct Piece<bf16, 8> {
  typedef uint4 Raw;
  static __device__ __forceinline__ Raw load(const bf16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
  static __device__ __forceinline__ void unpack(const Raw& r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ void store(bf16* p, const float* v) {
    uint4 r;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = r;
  }
};
template <> struct Piece<float, 4> {
  typedef float4 Raw;
  static __device__ __forceinline__ Raw load(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
  static __device__ __forceinline__ void unpack(const Raw& r, float* v) { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
  static __device__ __forceinline__ void store(float* p, const float* v) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
};
// columns c ... of the weight, zeros where there are none
template <int VEC, bool SHIFT, typename W> __device__ __forceinline__ void load_weight(const W* w, int c, int width, float* v) {
  w += c;
  if constexpr (SHIFT) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = c + j >= 0 && c + j < width ? to_f(w[j]) : 0.f;
  } else if constexpr (sizeof(W) == 2) {
    Piece<bf16, 8>::unpack(Piece<bf16, 8>::load(w), v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) Piece<float, 4>::unpack(Piece<float, 4>::load(w + i), v + i);
  }
}
// Codes of a row's columns c ... Shifted ones are stored in twos, from the second on where the first lies on an odd address, and only those at
// a row's ends are looked at one by one: 4096 rows of 4095 columns in bf16 34.7 -> 29.0 us, of 8185 68.8 -> 54.6; in fp32 no change (12289 x
// 1001 25). To put them together into words with the next lane's takes longer, 72 and 78 us, since a warp's ends are then left over.
template <int VEC, bool SHIFT> __device__ __forceinline__ void store_codes(uint8_t* p, int c, int width, const float* v) {
  uint32_t w[VEC / 4];
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | hi << 16;
  }
  auto code = [&](int j) { return w[j / 4] >> 8 * (j % 4); };
  p += c;
  if constexpr (!SHIFT) {
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  } else if (c < 0 || c + VEC > width) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (c + j >= 0 && c + j < width) p[j] = (uint8_t)code(j);
  } else if (reinterpret_cast<uintptr_t>(p) & 1) {
    p[0] = (uint8_t)code(0);
#pragma unroll
    for (int j = 1; j < VEC - 1; j += 2) *reinterpret_cast<uint16_t*>(p + j) = (uint16_t)(j % 4 == 3 ? __funnelshift_r(w[j / 4], w[(j + 1) / 4], 24) : code(j));
    p[VEC - 1] = (uint8_t)code(VEC - 1);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) *reinterpret_cast<uint16_t*>(p + j) = (uint16_t)code(j);
  }
}

// How rows lie. In all three a thread has the same columns of a row, so that a row's sums have the same bits:
//   kAligned  whole pieces of 16 bytes
//   kShifted  rows of any width one after the other: their pieces start up to VEC - 1 elements in front of the row. A group's rows are a
//             multiple of VEC apart, so that all of them, and with them the columns of its threads, are shifted alike; what a piece
//             holds of the rows beside is left out
//   kSingle   anything else, element by element
enum Kind { kAligned, kShifted, kSingle };

// A thread's pieces of its next AT - 1 rows come ahead of it into shared memory, where 16 bytes of a thread lie beside the next thread's:
// it reads what it asked for itself, so nothing synchronises. Single elements are read when their row's turn comes.
template <typename T, int VEC, int NV, int NT, int KIND>
struct Rows {
  typedef Piece<T, VEC> P;
  static constexpr int AT = NV > 2 ? 2 : NV == 2 && NT == 2 ? 3 : 4;         // what a thousand threads' share of shared memory holds
  static constexpr int THREAD = KIND == kSingle ? 0 : AT * NT * NV * 16;       // bytes of shared memory
  uint8_t* ring;
  __device__ __forceinline__ explicit Rows(uint8_t* shared) : ring(shared + threadIdx.x * 16) {}
  __device__ __forceinline__ uint8_t* slot(int stage, int tensor, int k) const { return ring + ((stage * NT + tensor) * NV + k) * (int)blockDim.x * 16; }
  // tensors' columns c0 + k * group * VEC ... of a row; `left`: elements from its first one to the tensor's end
  __device__ __forceinline__ void request(int stage, const T* const* from, bool there, int c0, int group, int width, long long left) {
    if constexpr (KIND != kSingle) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = c0 + k * group * VEC;
          if (there && from[t] != nullptr && c < width) {
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(slot(stage, t, k));
            if (KIND == kShifted) {
              const int bytes = left - c < VEC ? (int)(left - c) * (int)sizeof(T) : 16;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from[t] + c), "r"(bytes) : "memory");
            } else {
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from[t] + c) : "memory");
            }
          }
        }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  __device__ __forceinline__ void arrived() const {
    if constexpr (KIND != kSingle) asm volatile("cp.async.wait_group %0;" ::"n"(AT - 1) : "memory");
  }
  __device__ __forceinline__ void all_arrived() const {
    if constexpr (KIND != kSingle) asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  // columns c ... of the current row, zeros in those that are not the row's
  __device__ __forceinline__ void read(int stage, int tensor, int k, const T* from, int c, int width, float* v) const {
    if constexpr (KIND == kSingle) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = c + j >= 0 && c + j < width ? to_f(from[c + j]) : 0.f;
    } else {
      P::unpack(*reinterpret_cast<const typename P::Raw*>(slot(stage, tensor, k)), v);
      if (KIND == kShifted && (c < 0 || c + VEC > width)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = c + j >= 0 && c + j < width ? v[j] : 0.f;
      }
    }
  }
  // to rows one after the other, of which the first starts on 16 bytes
  static __device__ __forceinline__ void write(T* to, int c, int width, const float* v) {
    if (KIND == kAligned || (c >= 0 && c + VEC <= width)) {
      P::store(to + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c + j >= 0 && c + j < width) to[c + j] = from_f<T>(v[j]);
    }
  }
};

// Two values from all threads of a row's group (`group` threads, a multiple of 32), in one exchange. `shared`: a pair per warp, used by one
// exchange after another in turns of two.
template <class Op, class Op2>
__device__ __forceinline__ float2 group_all(float2 v, int group, float2 (*shared)[16], int& turn, Op op, Op2 op2) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x = op(v.x, __shfl_xor_sync(0xffffffffu, v.x, o));
    v.y = op2(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
  }
  if (group == 32) return v;
  float2* s = shared[turn ^= 1];
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  const int first = threadIdx.x / group * (group / 32);
  v = s[first];
  for (int w = 1; w < group / 32; ++w) {
    const float2 u = s[first + w];
    v.x = op(v.x, u.x);
    v.y = op2(v.y, u.y);
  }
  return v;
}

template <typename T, typename W, int VEC, int NV, int KIND, bool QUANT>
__global__ void __launch_bounds__(512) norm_kernel(const NormRows p, T* __restrict__ y, uint8_t* __restrict__ codes, long long codes_ld, float* __restrict__ scales,
                                                    const int group) {
  constexpr bool SHIFT = KIND != kAligned;
  extern __shared__ __align__(16) uint8_t ahead[];
  __shared__ float2 shared[2][16];
  pdl_sync();
  const int beside = blockDim.x / group, mine = threadIdx.x % group;
  const long long step = (long long)gridDim.x * beside;
  long long row = (long long)blockIdx.x * beside + threadIdx.x / group;
  const int c0 = mine * VEC - (SHIFT ? (int)(row * p.width % VEC) : 0);        // this thread's first column
  const float inv_width = 1.0f / p.width;
  int turn = 0;
  float w[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = c0 + k * group * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[k][j] = 1.0f;
    if (p.weight != nullptr && c < p.width) load_weight<VEC, SHIFT>(static_cast<const W*>(p.weight), c, p.width, w[k]);
  }
  typedef Rows<T, VEC, NV, 2, KIND> R;
  R rows(ahead);
  constexpr int AT = R::AT;
  struct From { const T* at[2]; };
  auto from = [&](long long r) {
    return From{{static_cast<const T*>(p.x) + r * p.x_ld, p.res != nullptr ? static_cast<const T*>(p.res) + r * p.res_ld : nullptr}};
  };
  auto request = [&](int stage, long long r) { rows.request(stage, from(r).at, r < p.rows, c0, group, p.width, (p.rows - r) * p.width); };
#pragma unroll
  for (int k = 0; k < AT - 1; ++k) request(k, row + k * step);
  int stage = 0;
  // every thread goes as often as the block's first group: the sums synchronise
  for (long long base = (long long)blockIdx.x * beside; base < p.rows; base += step, row += step, stage = (stage + 1) % AT) {
    const bool there = row < p.rows;
    request((stage + AT - 1) % AT, row + (AT - 1) * step);
    rows.arrived();
    const From at = from(row);
    float v[NV][VEC];
    float q = 0.f, most = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * group * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] = 0.f;
      if (there && c < p.width) {
        rows.read(stage, 0, k, at.at[0], c, p.width, v[k]);
        if (p.res != nullptr) {
          float r[VEC];
          rows.read(stage, 1, k, at.at[1], c, p.width, r);
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[k][j] = to_f(from_f<T>(v[k][j] + r[j]));
          R::write(static_cast<T*>(p.sum) + row * p.width, c, p.width, v[k]);
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        q = fmaf(v[k][j], v[k][j], q);
        if (QUANT) most = max_nan(most, fabsf(v[k][j] * w[k][j]));
      }
    }
    float rstd = 1.0f;
    if (QUANT || p.weight != nullptr) {
      const float2 r = group_all(make_float2(q, most), group, shared, turn, Add(), Max());
      if (p.weight != nullptr) rstd = rsqrtf(r.x * inv_width + p.eps);
      most = r.y;
    }
    // the largest size of the products is found beside the sum of squares: rstd, which they share, is one more factor of it
    const float scale = most * rstd / kE4m3Max, inv = scale == 0.f ? 0.f : rstd / scale;
    if (QUANT && there && mine == 0) scales[row] = scale;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * group * VEC;
      const float factor = QUANT ? inv : rstd;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] = v[k][j] * factor * w[k][j];
      if (there && c < p.width) {
        if (QUANT) store_codes<VEC, SHIFT>(codes + row * codes_ld, c, p.width, v[k]);
        else R::write(y + row * p.width, c, p.width, v[k]);
      }
    }
  }
}

// Gradients of rows and, in part[block], of the weight over the block's rows.
template <typename T, typename W, int VEC, int NV, int KIND>
__global__ void __launch_bounds__(512, VEC * NV <= 8 ? 2 : 1) norm_bwd_kernel(const NormGrad p, const int group) {
  constexpr bool SHIFT = KIND != kAligned;
  extern __shared__ __align__(16) uint8_t ahead[];
  __shared__ float2 shared[2][16];
  pdl_sync();
  const int beside = blockDim.x / group, mine = threadIdx.x % group;
  const long long step = (long long)gridDim.x * beside;
  long long row = (long long)blockIdx.x * beside + threadIdx.x / group;
  const int c0 = mine * VEC - (SHIFT ? (int)(row * p.width % VEC) : 0);        // this thread's first column
  const float inv_width = 1.0f / p.width;
  int turn = 0;
  float w[NV][VEC], dw[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = c0 + k * group * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[k][j] = dw[k][j] = 0.f;
    if (c < p.width) load_weight<VEC, SHIFT>(static_cast<const W*>(p.weight), c, p.width, w[k]);
  }
  typedef Rows<T, VEC, NV, 3, KIND> R;
  R rows(ahead);
  constexpr int AT = R::AT;
  struct From { const T* at[3]; };
  auto from = [&](long long r) {
    return From{{static_cast<const T*>(p.s) + r * p.s_ld, static_cast<const T*>(p.dy) + r * p.dy_ld, p.ds != nullptr ? static_cast<const T*>(p.ds) + r * p.ds_ld : nullptr}};
  };
  auto request = [&](int stage, long long r) { rows.request(stage, from(r).at, r < p.rows, c0, group, p.width, (p.rows - r) * p.width); };
#pragma unroll
  for (int k = 0; k < AT - 1; ++k) request(k, row + k * step);
  int stage = 0;
  for (long long base = (long long)blockIdx.x * beside; base < p.rows; base += step, row += step, stage = (stage + 1) % AT) {
    const bool there = row < p.rows;
    request((stage + AT - 1) % AT, row + (AT - 1) * step);
    rows.arrived();
    const From at = from(row);
    float s[NV][VEC], g[NV][VEC];
    float q = 0.f, d = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * group * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[k][j] = g[k][j] = 0.f;
      if (there && c < p.width) {
        rows.read(stage, 0, k, at.at[0], c, p.width, s[k]);
        rows.read(stage, 1, k, at.at[1], c, p.width, g[k]);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        q = fmaf(s[k][j], s[k][j], q);
        d = fmaf(s[k][j] * g[k][j], w[k][j], d);
      }
    }
    const float2 r = group_all(make_float2(q, d), group, shared, turn, Add(), Add());
    const float rstd = rsqrtf(r.x * inv_width + p.eps), along = r.y * rstd * inv_width * rstd;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * group * VEC;
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] = 0.f;
      if (p.ds != nullptr && there && c < p.width) rows.read(stage, 2, k, at.at[2], c, p.width, o);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float n = s[k][j] * rstd;
        dw[k][j] = fmaf(g[k][j], n, dw[k][j]);
        o[j] = fmaf(g[k][j] * w[k][j], rstd, fmaf(-n, along, o[j]));
      }
      if (there && c < p.width) R::write(static_cast<T*>(p.dx) + row * p.width, c, p.width, o);
    }
  }
  float* part = p.part + (long long)blockIdx.x * p.width;
  rows.all_arrived();
  if (beside == 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * group * VEC;
      if (c < p.width)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!SHIFT || (c + j >= 0 && c + j < p.width)) part[c + j] = dw[k][j];
    }
  } else {
    float* sums = reinterpret_cast<float*>(ahead);         // [group][width], where the rows were
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * group * VEC;
      if (c < p.width)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!SHIFT || (c + j >= 0 && c + j < p.width)) sums[threadIdx.x / group * p.width + c + j] = dw[k][j];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
      float sum = sums[c];
      for (int b = 1; b < beside; ++b) sum += sums[b * p.width + c];
      part[c] = sum;
    }
  }
}

// dw = the sum of the parts: 32 columns a block, its warps a share of the parts each.
constexpr int kSumWarps = 32;
template <typename W>
__global__ void __launch_bounds__(32 * kSumWarps) norm_dw_sum_kernel(const float* __restrict__ part, W* __restrict__ dw, int parts, int width) {
  __shared__ float shared[kSumWarps][33];
  pdl_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < width)
#pragma unroll 8
    for (int k = warp; k < parts; k += kSumWarps) sum += part[(long long)k * width + c];
  shared[warp][lane] = sum;
  __syncthreads();
  sum = shared[lane][warp];                  // column `warp` of the block, part `lane`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0 && blockIdx.x * 32 + warp < width) dw[blockIdx.x * 32 + warp] = from_f<W>(sum);
}

// ------------------------------------------------------------------------------------------------ wide rows
// Wide rows. A block per row; QUANT: rows leave in 8 bits.
template <typename T, typename W, bool QUANT>
__global__ void __launch_bounds__(kThreads) wide_norm_kernel(const NormRows p, T* __restrict__ y, uint8_t* __restrict__ codes, long long codes_ld,
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
__global__ void __launch_bounds__(kThreads) wide_norm_dx_kernel(const NormGrad p, float* __restrict__ rstds) {
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
__global__ void __launch_bounds__(kThreads) wide_norm_dw_kernel(const NormGrad p, const float* __restrict__ rstds, float* __restrict__ part, int parts) {
  pdl_sync();
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= p.width) return;
  float sum = 0.f;
  for (long long row = blockIdx.y; row < p.rows; row += parts)
    sum += to_f(static_cast<const T*>(p.dy)[row * p.dy_ld + c]) * to_f(static_cast<const T*>(p.s)[row * p.s_ld + c]) * rstds[row];
  part[(long long)blockIdx.y * p.width + c] = sum;
}

// ------------------------------------------------------------------------------------------------ host
// How many pieces a thread holds and how many threads share a row. One piece where a row's latency counts; where the rows alone fill the SMs
// two, or four where a warp has the row to itself then (no barrier: 20000 x 300 in fp32 13.3 -> 11.6 us, in 8 bits 15.9 -> 13.4; wider
// rows lose some: 12288 x 1024 in 8 bits 27.1 -> 28.8). Backward in fp32 four: 4096 x 4096 50.7 -> 47.1 us, 20000 x 300 25.5 -> 17.6;
// in bf16 their 32 columns a thread do not fit the registers. Groups are whole warps rather than powers of two: 4096 rows in bf16 of 4095
// columns 31.9 / 69.6 -> 26.5 / 55.0 us, of 2047 16.9 / 35.6 -> 16.2 / 26.0, 3000 in fp32 22.5 / 29.2 -> 19.6 / 27.8; 6001 forward 32.0 -> 33.9.
struct Layout { int pieces, group; };       // pieces 0: the row does not fit
Layout layout_of(long long rows, int width, int vec, bool backward) {
  const int all = width % vec == 0 ? width / vec : (width + 2 * vec - 2) / vec;
  auto group_for = [&](int pieces) {
    const int warps = (all + 32 * pieces - 1) / (32 * pieces);
    return 32 * (warps < 16 ? warps : 16);
  };
  int pieces = 1;
  if (rows >= 4LL * sm_count()) pieces = backward ? (vec == 4 ? 4 : 2) : all > 64 && all <= 128 ? 4 : 2;
  while (pieces < 4 && group_for(pieces) * pieces < all) pieces *= 2;
  const int group = group_for(pieces);
  return group * pieces < all ? Layout{0, 0} : Layout{pieces, group};
}
int block_of(int group) { return group < 256 ? 256 / group * group : group; }

bool aligned(const void* p, long long ld, int bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * bytes % 16 == 0; }
Kind kind_of(const NormRows& p, const void* y) {
  const int size = p.bf16 ? 2 : 4;
  auto fits = [&](int bytes) {
    return aligned(p.x, p.x_ld, bytes) && aligned(p.res, p.res_ld, bytes) && aligned(p.sum, p.width, bytes) && aligned(y, p.width, bytes);
  };
  if (fits(size) && p.width * size % 16 == 0 && aligned(p.weight, 0, 1)) return kAligned;
  return fits(16) && p.x_ld == p.width && (p.res == nullptr || p.res_ld == p.width) ? kShifted : kSingle;
}
Kind kind_of(const NormGrad& p) {
  const int size = p.bf16 ? 2 : 4;
  auto fits = [&](int bytes) {
    return aligned(p.s, p.s_ld, bytes) && aligned(p.dy, p.dy_ld, bytes) && aligned(p.ds, p.ds_ld, bytes) && aligned(p.dx, p.width, bytes);
  };
  if (fits(size) && p.width * size % 16 == 0 && aligned(p.weight, 0, 1)) return kAligned;
  return fits(16) && p.s_ld == p.width && p.dy_ld == p.width && (p.ds == nullptr || p.ds_ld == p.width) ? kShifted : kSingle;
}
// Blocks whose groups walk along rows that are shifted alike.
long long walking(long long blocks, long long most, int beside, int vec) {
  if (blocks <= most) return blocks;
  while (most > 1 && most * beside % vec != 0) --most;
  return most;
}

// More shared memory than a kernel has by itself has to be asked for, once.
cudaError_t allow(const void* kernel, size_t smem) {
  if (smem <= 40 * 1024) return cudaSuccess;
  static std::mutex mutex;
  static std::set<const void*> asked;
  const std::lock_guard<std::mutex> lock(mutex);
  if (asked.count(kernel)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  if (e == cudaSuccess) asked.insert(kernel);
  return e;
}

template <typename T, typename W, bool QUANT, int KIND>
cudaError_t forward_rows(const NormRows& p, const Layout& l, void* y, void* codes, long long codes_ld, float* scales, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const int block = block_of(l.group), beside = block / l.group;
  const long long blocks = walking((p.rows + beside - 1) / beside, (long long)sm_count() * (l.pieces * VEC <= 8 ? 2048 : 1024) / block, beside, VEC);
  auto with = [&](auto kernel, int thread) {
    const size_t smem = (size_t)thread * block;
    const cudaError_t e = allow(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)blocks), dim3(block), smem, st, p, static_cast<T*>(y), static_cast<uint8_t*>(codes), codes_ld, scales, l.group);
  };
  if (l.pieces == 1) return with(norm_kernel<T, W, VEC, 1, KIND, QUANT>, Rows<T, VEC, 1, 2, KIND>::THREAD);
  if (l.pieces == 2) return with(norm_kernel<T, W, VEC, 2, KIND, QUANT>, Rows<T, VEC, 2, 2, KIND>::THREAD);
  return with(norm_kernel<T, W, VEC, 4, KIND, QUANT>, Rows<T, VEC, 4, 2, KIND>::THREAD);
}
template <typename T, typename W, bool QUANT>
cudaError_t forward(const NormRows& p, void* y, void* codes, long long codes_ld, float* scales, cudaStream_t st) {
  if (p.rows <= 0) return cudaSuccess;
  const Kind kind = kind_of(p, y);
  const Layout l = layout_of(p.rows, p.width, 16 / sizeof(T), false);
  if (l.pieces != 0) {
    if (kind == kAligned) return forward_rows<T, W, QUANT, kAligned>(p, l, y, codes, codes_ld, scales, st);
    if (kind == kShifted) return forward_rows<T, W, QUANT, kShifted>(p, l, y, codes, codes_ld, scales, st);
    return forward_rows<T, W, QUANT, kSingle>(p, l, y, codes, codes_ld, scales, st);
  }
  const long long most = 8LL * sm_count();
  return launch_pdl(wide_norm_kernel<T, W, QUANT>, dim3((unsigned)(p.rows < most ? p.rows : most)), dim3(kThreads), 0, st, p, static_cast<T*>(y),
                    static_cast<uint8_t*>(codes), codes_ld, scales);
}
template <bool QUANT>
cudaError_t forward_of(const NormRows& p, void* y, void* codes, long long codes_ld, float* scales, cudaStream_t st) {
  if (!p.bf16) return p.weight_bf16 ? cudaErrorInvalidValue : forward<float, float, QUANT>(p, y, codes, codes_ld, scales, st);
  return p.weight_bf16 ? forward<bf16, bf16, QUANT>(p, y, codes, codes_ld, scales, st) : forward<bf16, float, QUANT>(p, y, codes, codes_ld, scales, st);
}

constexpr int kWideParts = 64;
constexpr int kThreadsBack = 512;            // on an SM, twice as many where a thread has 8 columns at most

Layout layout_back(const NormGrad& p) { return layout_of(p.rows, p.width, p.bf16 ? 8 : 4, true); }
long long blocks_back(const NormGrad& p, const Layout& l) {
  const int block = block_of(l.group), beside = block / l.group, vec = p.bf16 ? 8 : 4;
  const long long most = (long long)sm_count() * (kThreadsBack / block) * (l.pieces * vec <= 8 ? 2 : 1);
  return walking((p.rows + beside - 1) / beside, most, beside, vec);
}

template <typename T, typename W, int KIND>
cudaError_t backward_rows(const NormGrad& p, const Layout& l, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const int block = block_of(l.group), beside = block / l.group;
  auto with = [&](auto kernel, int thread) {
    const size_t joined = beside > 1 ? (size_t)beside * p.width * sizeof(float) : 0, ahead = (size_t)thread * block, smem = joined > ahead ? joined : ahead;
    const cudaError_t e = allow(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)blocks_back(p, l)), dim3(block), smem, st, p, l.group);
  };
  if (l.pieces == 1) return with(norm_bwd_kernel<T, W, VEC, 1, KIND>, Rows<T, VEC, 1, 3, KIND>::THREAD);
  if (l.pieces == 2) return with(norm_bwd_kernel<T, W, VEC, 2, KIND>, Rows<T, VEC, 2, 3, KIND>::THREAD);
  return with(norm_bwd_kernel<T, W, VEC, 4, KIND>, Rows<T, VEC, 4, 3, KIND>::THREAD);
}
template <typename T, typename W>
cudaError_t backward(const NormGrad& p, int* launched, cudaStream_t st) {
  const Kind kind = kind_of(p);
  const Layout l = layout_back(p);
  int parts = 0;
  cudaError_t e = cudaSuccess;
  *launched = 1;
  if (p.rows > 0 && l.pieces != 0) {
    parts = (int)blocks_back(p, l);
    *launched = 2;
    if (kind == kAligned) e = backward_rows<T, W, kAligned>(p, l, st);
    else if (kind == kShifted) e = backward_rows<T, W, kShifted>(p, l, st);
    else e = backward_rows<T, W, kSingle>(p, l, st);
  } else if (p.rows > 0) {
    parts = kWideParts;
    *launched = 3;
    float* rstds = p.part + (long long)parts * p.width;
    const long long most = 8LL * sm_count();
    e = launch_pdl(wide_norm_dx_kernel<T, W>, dim3((unsigned)(p.rows < most ? p.rows : most)), dim3(kThreads), 0, st, p, rstds);
    if (e == cudaSuccess)
      e = launch_pdl(wide_norm_dw_kernel<T>, dim3((p.width + kThreads - 1) / kThreads, parts), dim3(kThreads), 0, st, p, rstds, p.part, parts);
  }
  if (e != cudaSuccess) return e;
  return launch_pdl(norm_dw_sum_kernel<W>, dim3((p.width + 31) / 32), dim3(32 * kSumWarps), 0, st, p.part, static_cast<W*>(p.dw), parts, p.width);
}

}  // namespace

cudaError_t rms_norm_fwd(const NormRows& p, void* y, cudaStream_t st) { return forward_of<false>(p, y, nullptr, 0, nullptr, st); }
cudaError_t rms_norm_8bit(const NormRows& p, void* codes, long long codes_ld, float* scales, cudaStream_t st) {
  return forward_of<true>(p, nullptr, codes, codes_ld, scales, st);
}
long long rms_norm_bwd_floats(const NormGrad& p) {
  const Layout l = layout_back(p);
  return l.pieces != 0 ? blocks_back(p, l) * p.width : (long long)kWideParts * p.width + p.rows;       // the rows' rstd behind the sums
}
cudaError_t rms_norm_bwd(const NormGrad& p, int* launched, cudaStream_t st) {
  if (!p.bf16) return p.weight_bf16 ? cudaErrorInvalidValue : backward<float, float>(p, launched, st);
  return p.weight_bf16 ? backward<bf16, bf16>(p, launched, st) : backward<bf16, float>(p, launched, st);
}

}  // namespace adb200
