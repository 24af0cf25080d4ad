// Product of rows in 8 bits with a scale each: y = (codes . weight_codes^T) * scales * weight_scales + bias, on tcgen05.mma kind::f8f6f4.
// e4m3 products and their fp32 sums come out of the tensor cores; the scales, which are constant along the contraction, are applied once to
// the finished sum, and the bf16 result is the only rounding.
//
// Two kernels, with the roles of the bf16 products (one warp issues TMA copies, one the MMAs, the others drain the accumulator); a K block
// is 128 bytes, 128 codes here, so that tiles, swizzle and descriptors are those of 64 bf16 values:
//
//   pairs   256 x 256 tiles on two SMs (cta_group::2), persistent, two accumulators: prompts, bound by the tensor cores
//   tiles   the weight's rows are the MMA's 128 rows and 16 to 128 rows of codes its columns, so that a few tokens fill a tile;
//           the contraction is split over a cluster where the tiles leave SMs idle, and summed through distributed shared memory in a
//           fixed order: decoding steps, bound by reading the weight
//
// Measured (B200, replayed back to back, operands in the L2 where they fit; rows x contraction x columns): 8192 x 4096 x 4096 97 us, 2846 TFLOP/s,
// 0.85 of twice the bf16 burst rate; 1024 x 4096 x 4096 16; 8192 x 512 x 4096 25 us, of which memory and tensor cores need 11 and 10 each
// (44 us when a lane drained a row of its own instead of fragments); 8 x 2048 x 8192 5.2 us (the weight's bytes from
// memory alone would take 2.6).
#include "gemm_8bit.h"

#include <cuda.h>
#include <cuda_bf16.h>

#include <array>
#include <mutex>

#include "gemm_epilogue.cuh"
#include "pair_tcgen05.cuh"
#include "pdl.cuh"
#include "sm_count.h"
#include "tcgen05_common.cuh"

namespace adb200 {
namespace {

using namespace tc;

constexpr int KB = 128;                      // codes of a K block: one swizzled row of 128 bytes
constexpr int kMmaK = 32;                    // codes of one MMA
constexpr int kRowsBytes = 128 * KB;         // 128 rows of a K block

// Instruction descriptor of kind::f8f6f4: fp32 sums of e4m3 products, both operands K-major.
__device__ __forceinline__ uint32_t make_idesc8(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

__device__ __forceinline__ void umma8(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma8_pair(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void give_up(volatile int* abort_flag, int* error, int code) {
  *abort_flag = 1;
  if (error != nullptr) atomicExch(error, code);
}
// Four values of a vector of n, zeros past its end. `i` is a multiple of 4, the vector's base on 16 bytes.
__device__ __forceinline__ float4 four_of(const float* v, int i, int n) {
  if (i + 4 <= n) return __ldg(reinterpret_cast<const float4*>(v + i));
  return make_float4(i < n ? v[i] : 0.f, i + 1 < n ? v[i + 1] : 0.f, i + 2 < n ? v[i + 2] : 0.f, 0.f);
}

// Two of them from an even place on.
__device__ __forceinline__ float2 two_of(const float* v, int i, int n) {
  if (i + 2 <= n) return __ldg(reinterpret_cast<const float2*>(v + i));
  return make_float2(i < n ? v[i] : 0.f, 0.f);
}

// ------------------------------------------------------------------------------------------------ tiles
constexpr int kTileThreads = 192;            // warps: TMA, MMA, four that drain
template <int BN> struct TileCfg {
  static constexpr int STAGE = kRowsBytes + BN * KB;
  static constexpr int STAGES = BN >= 128 ? 6 : 8;
  static constexpr int RING = STAGES * STAGE;          // the fp32 sums [BN][128] are laid over it: 512 BN bytes
  static constexpr int SMEM = RING + 1024 /*align*/ + 256 /*barriers*/;
  static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  static_assert(RING >= BN * 128 * 4, "sums in the ring");
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// This CTA's share of the tile's tokens: sums over the S partial sums, scaled and stored, four outputs at a time.
template <int BN, int S>
__device__ __forceinline__ void sum_and_store(const Gemm8Args& a, uint32_t sums, uint32_t rank, int m0, int n0) {
  const int tokens = min(BN, a.M - m0);
  const int t0 = (int)rank * tokens / S, t1 = ((int)rank + 1) * tokens / S;
  uint32_t peer[S];
#pragma unroll
  for (int s = 0; s < S; ++s) peer[s] = S == 1 ? sums : map_to_cta(sums, (uint32_t)s);
  const int col = n0 + 4 * ((int)threadIdx.x & 31);
  if (col >= a.N) return;
  const float4 sw = four_of(a.weight_scales, col, a.N);
  const float4 bias = a.bias != nullptr ? four_of(a.bias, col, a.N) : make_float4(0.f, 0.f, 0.f, 0.f);
  const bool whole = (a.N & 3) == 0;
#pragma unroll 2
  for (int t = t0 + ((int)threadIdx.x >> 5); t < t1; t += kTileThreads / 32) {
    const uint32_t off = (uint32_t)(t * 512 + ((int)threadIdx.x & 31) * 16);
    float4 x[S];
#pragma unroll
    for (int s = 0; s < S; ++s) x[s] = ld_cluster_f4(peer[s] + off);
    const float sx = __ldg(a.scales + m0 + t);
    float4 v = x[0];
#pragma unroll
    for (int s = 1; s < S; ++s) { v.x += x[s].x; v.y += x[s].y; v.z += x[s].z; v.w += x[s].w; }
    v.x = fmaf(v.x, sx * sw.x, bias.x); v.y = fmaf(v.y, sx * sw.y, bias.y); v.z = fmaf(v.z, sx * sw.z, bias.z); v.w = fmaf(v.w, sx * sw.w, bias.w);
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.y) + (long long)(m0 + t) * a.N + col;
    if (whole) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
    } else {
      dst[0] = __float2bfloat16(v.x);
      if (col + 1 < a.N) dst[1] = __float2bfloat16(v.y);
      if (col + 2 < a.N) dst[2] = __float2bfloat16(v.z);
      if (col + 3 < a.N) dst[3] = __float2bfloat16(v.w);
    }
  }
}

template <int BN>
__global__ void __launch_bounds__(kTileThreads, 1)
gemm8_tile_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const Gemm8Args a, const int split) {
  using C = TileCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::RING);
  uint64_t* empty = full + C::STAGES;
  uint64_t* done = empty + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = split > 1 ? cluster_ctarank() : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_sync();

  const int tiles_m = (a.M + BN - 1) / BN;
  const int t = (int)(blockIdx.x / (unsigned)split);
  const int m0 = t % tiles_m * BN, n0 = t / tiles_m * 128;
  const int num_kb = (a.K + KB - 1) / KB;
  const int kb0 = (int)((long long)num_kb * rank / split), kb1 = (int)((long long)num_kb * (rank + 1) / split);

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0, issued = 0; uint32_t phase = 0; bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) { ok = false; break; }
        ++issued;
        uint8_t* dst = smem + stage * C::STAGE;
        mbar_expect_tx(&full[stage], C::STAGE);
        load_2d(dst, &tm_w, &full[stage], kb * KB, n0);
        load_2d(dst + kRowsBytes, &tm_x, &full[stage], kb * KB, m0);
        if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
      }
      if (!ok) give_up(abort_flag, a.error, 81);
      if (*abort_flag) {                                  // copies in flight land before the ring is written over or the CTA leaves
        for (int i = issued > C::STAGES ? issued - C::STAGES : 0; i < issued; ++i) {
          const long long w0 = clock64();
          while (!mbar_try(&full[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u) && clock64() - w0 < 20000000LL) {}
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = make_idesc8(128, BN);
      int stage = 0; uint32_t phase = 0; bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t w_addr = smem_u32(smem + stage * C::STAGE), x_addr = w_addr + kRowsBytes;
#pragma unroll
        for (int k = 0; k < KB / kMmaK; ++k)
          umma8(tmem, make_desc(w_addr + k * kMmaK, 16, 1024), make_desc(x_addr + k * kMmaK, 16, 1024), idesc, kb != kb0 || k != 0 ? 1u : 0u);
        umma_commit(&empty[stage]);
        if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
      }
      if (ok) umma_commit(done);
      else give_up(abort_flag, a.error, 82);
    }
  } else {
    // every MMA of this CTA has completed when `done` flips: the ring is idle and takes the sums, a token's 128 outputs after the other's
    const int q = warp & 3;
    if (mbar_wait(done, 0, abort_flag)) {
      tc_fence_after();
      const uint32_t t_row = tmem + ((uint32_t)(q * 32) << 16);
      const uint32_t dst = smem_u32(smem) + (uint32_t)((q * 32 + lane) * 4);
      const int tokens = min(BN, a.M - m0);
#pragma unroll 1
      for (int c = 0; c < BN && c < tokens; c += 16) {
        float v[16];
        __syncwarp();
        tmem_ld16(t_row + c, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) sts1(dst + (uint32_t)((c + j) * 512), __float_as_uint(v[j]));
      }
    } else if (lane == 0) {
      give_up(abort_flag, a.error, 83);
    }
  }

  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (split > 1) cluster_sync_all();                       // all partial sums of the cluster are in shared memory
  const uint32_t sums = smem_u32(smem);
  switch (split) {
    case 1: sum_and_store<BN, 1>(a, sums, rank, m0, n0); break;
    case 2: sum_and_store<BN, 2>(a, sums, rank, m0, n0); break;
    case 3: sum_and_store<BN, 3>(a, sums, rank, m0, n0); break;
    case 4: sum_and_store<BN, 4>(a, sums, rank, m0, n0); break;
    case 5: sum_and_store<BN, 5>(a, sums, rank, m0, n0); break;
    case 6: sum_and_store<BN, 6>(a, sums, rank, m0, n0); break;
    case 7: sum_and_store<BN, 7>(a, sums, rank, m0, n0); break;
    default: sum_and_store<BN, 8>(a, sums, rank, m0, n0);
  }
  __syncwarp();
  if (split > 1) cluster_sync_all();                       // nobody leaves while a peer still reads its sums
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ pairs
// As the bf16 product on SM pairs: each CTA stages its half of both operands, the leader issues the MMAs, each CTA drains its own 128 rows.
constexpr int P_BN = 256;
constexpr int P_STAGE = 2 * kRowsBytes;
constexpr int P_STAGES = 5;
constexpr int P_EPI_WARPS = 8;               // two per TMEM lane quarter, 128 columns each
constexpr int P_THREADS = 64 + 32 * P_EPI_WARPS;
constexpr int P_STAGING = P_EPI_WARPS * 8192;          // two boxes of 32 rows x 64 columns per warp
constexpr int P_SMEM = P_STAGES * P_STAGE + P_STAGING + 1024 /*align*/ + 256 /*barriers*/;

__global__ void __launch_bounds__(P_THREADS, 1)
gemm8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_y, const Gemm8Args a,
                  const int store_boxes) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + P_STAGES * P_STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + P_STAGING);
  uint64_t* empty = full + P_STAGES;
  uint64_t* tfull = empty + P_STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();               // 0 = leader
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < P_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&tfull[s], 1); mbar_init(&tempty[s], 2 * P_EPI_WARPS); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * P_BN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                    // both CTAs' barriers exist before anything is signalled across
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_sync();

  const int tiles_m = (a.M + 255) / 256, tiles_n = (a.N + P_BN - 1) / P_BN;
  const long long total = (long long)tiles_m * tiles_n;
  const int num_kb = (a.K + KB - 1) / KB;
  const long long pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0; uint32_t phase = 0; bool ok = true;
      for (long long t = pair; t < total && ok; t += pairs) {
        const int m0 = (int)(t % tiles_m) * 256 + (int)rank * 128, n0 = (int)(t / tiles_m) * P_BN + (int)rank * 128;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) { ok = false; break; }
          if (leader) mbar_expect_tx(&full[stage], 2 * P_STAGE);
          const uint32_t bar = map_to_cta(smem_u32(&full[stage]), 0);
          uint8_t* dst = smem + stage * P_STAGE;
          load_2d_pair(dst, &tm_x, bar, kb * KB, m0);
          load_2d_pair(dst + kRowsBytes, &tm_w, bar, kb * KB, n0);
          if (++stage == P_STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) give_up(abort_flag, a.error, 84);
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      const uint32_t idesc = make_idesc8(256, P_BN);
      int stage = 0; uint32_t phase = 0; int as = 0; uint32_t aphase = 0; bool ok = true;
      for (long long t = pair; t < total && ok; t += pairs) {
        if (!mbar_wait(&tempty[as], aphase ^ 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(as * P_BN);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t x_addr = smem_u32(smem + stage * P_STAGE), w_addr = x_addr + kRowsBytes;
#pragma unroll
          for (int k = 0; k < KB / kMmaK; ++k)
            umma8_pair(d, make_desc(x_addr + k * kMmaK, 16, 1024), make_desc(w_addr + k * kMmaK, 16, 1024), idesc, (kb | k) != 0 ? 1u : 0u);
          umma2_commit(smem_u32(&empty[stage]));
          umma2_commit(map_to_cta(smem_u32(&empty[stage]), 1));
          if (++stage == P_STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        umma2_commit(smem_u32(&tfull[as]));
        umma2_commit(map_to_cta(smem_u32(&tfull[as]), 1));
        if (++as == 2) { as = 0; aphase ^= 1; }
      }
      if (!ok) give_up(abort_flag, a.error, 85);
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;
    const uint32_t box = smem_u32(staging) + (uint32_t)(warp - 2) * 8192u;
    int as = 0; uint32_t aphase = 0; bool ok = true;
    for (long long t = pair; t < total && ok; t += pairs) {
      const int row0 = (int)(t % tiles_m) * 256 + (int)rank * 128 + q * 32, col0 = (int)(t / tiles_m) * P_BN + part * 128;
      // what belongs to the tile's rows and columns comes while the tile is still being multiplied: in the fragment layout a lane has columns
      // 8 k + 2 (lane % 4) and the one beside of the rows lane / 4 + 8 i
      float sx[4];
      float2 sw[16], bias[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) sx[i] = row0 + lane / 4 + 8 * i < a.M ? __ldg(a.scales + row0 + lane / 4 + 8 * i) : 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int col = col0 + 8 * k + 2 * (lane & 3);
        sw[k] = two_of(a.weight_scales, col, a.N);
        bias[k] = a.bias != nullptr ? two_of(a.bias, col, a.N) : make_float2(0.f, 0.f);
      }
      if (!mbar_wait(&tfull[as], aphase, abort_flag)) { ok = false; break; }
      tc_fence_after();
      const uint32_t t_w = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(as * P_BN + part * 128);
#pragma unroll
      for (int c = 0; c < 4; ++c) {                        // 32 columns; two of them fill a box
        uint32_t v[32];
        __syncwarp();
        tmem_ld_frag32(t_w + c * 32, v);
        if (c == 3) {                                      // this warp has read its part of the accumulator
          tc_fence_before();
          if (elect_one()) mbar_arrive_cluster(map_to_cta(smem_u32(&tempty[as]), 0));
        }
        const int col = col0 + c * 32;
        if ((c & 1) == 0) {                                // the box's last copy has left it
          if (elect_one()) bulk_wait_read<1>();
          __syncwarp();
        }
        const uint32_t buf = box + (uint32_t)(c >> 1) * 4096u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t r = (uint32_t)lane / 4 + 8 * i;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 w = sw[c * 4 + k], b = bias[c * 4 + k];
            const float x = __uint_as_float(v[(i / 2) * 16 + k * 4 + (i % 2) * 2]), y = __uint_as_float(v[(i / 2) * 16 + k * 4 + (i % 2) * 2 + 1]);
            const uint32_t chunk = (uint32_t)((c & 1) * 4 + k);
            sts1(buf + r * 128u + ((chunk ^ (r & 7)) << 4) + ((uint32_t)lane & 3u) * 4u, pack2(fmaf(x, sx[i] * w.x, b.x), fmaf(y, sx[i] * w.y, b.y)));
          }
        }
        if (c & 1) {
          const int first = col - 32;
          if (store_boxes) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (elect_one()) {
              if (first < a.N && row0 < a.M) store_2d(&tm_y, buf, first, row0);
              bulk_commit();
            }
          } else {                                         // rows that TMA cannot describe: two columns of a row per lane
            __syncwarp();
            for (int r = 0; r < 32 && row0 + r < a.M; ++r) {
              const uint32_t two = lds1(buf + (uint32_t)r * 128u + ((((uint32_t)lane >> 2) ^ (uint32_t)(r & 7)) << 4) + ((uint32_t)lane & 3u) * 4u);
              const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&two);
              __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.y) + (long long)(row0 + r) * a.N + first + 2 * lane;
              if (first + 2 * lane < a.N) dst[0] = h.x;
              if (first + 2 * lane + 1 < a.N) dst[1] = h.y;
            }
            __syncwarp();
          }
        }
      }
      if (++as == 2) { as = 0; aphase ^= 1; }
    }
    if (elect_one()) bulk_wait_read<0>();                  // this warp's copies have left its boxes
    if (!ok && lane == 0) give_up(abort_flag, a.error, 86);
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                      // neither CTA leaves, or frees TMEM, while the other still works
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * P_BN) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ host
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess) fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}
// [rows, cols] of `bytes` each, boxes of 128 bytes x `box_rows`, 128-byte swizzle, zeros outside
bool map_rows(CUtensorMap* m, CUtensorMapDataType type, int bytes, const void* base, long long rows, long long cols, long long ld_bytes, int box_rows) {
  const EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / bytes), (cuuint32_t)box_rows}, steps[2] = {1, 1};
  return fn(m, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN>
cudaError_t launch_tiles(const Gemm8Args& a, int split, cudaStream_t st) {
  static const cudaError_t configured = cudaFuncSetAttribute(gemm8_tile_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileCfg<BN>::SMEM);
  if (configured != cudaSuccess) return configured;
  CUtensorMap tm_x, tm_w;
  if (!map_rows(&tm_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.codes, a.M, a.K, a.codes_ld, BN) ||
      !map_rows(&tm_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.weight_codes, a.N, a.K, a.weight_ld, 128))
    return cudaErrorInvalidValue;
  const long long tiles = (long long)((a.M + BN - 1) / BN) * ((a.N + 127) / 128);
  if (tiles * split > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split));
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = TileCfg<BN>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, gemm8_tile_kernel<BN>, tm_x, tm_w, a, split);
}

cudaError_t launch_pairs(const Gemm8Args& a, cudaStream_t st) {
  static int max_pairs = 0;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(P_THREADS);
  cfg.dynamicSmemBytes = P_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  if (max_pairs == 0) {
    const cudaError_t e = cudaFuncSetAttribute(gemm8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P_SMEM);
    if (e != cudaSuccess) return e;
    int n = 0;                                             // SM pairs of one cluster sit in one GPC, so it can be fewer than SMs / 2
    cfg.gridDim = dim3((unsigned)(sm_count() & ~1));
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, gemm8_pair_kernel, &cfg) != cudaSuccess || n <= 0) { (void)cudaGetLastError(); n = sm_count() / 2; }
    max_pairs = n < sm_count() / 2 ? n : sm_count() / 2;
  }
  CUtensorMap tm_x, tm_w, tm_y;
  if (!map_rows(&tm_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.codes, a.M, a.K, a.codes_ld, 128) ||
      !map_rows(&tm_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.weight_codes, a.N, a.K, a.weight_ld, 128))
    return cudaErrorInvalidValue;
  const int boxes = a.N % 8 == 0;                          // rows of the result on 16-byte boundaries
  tm_y = tm_x;
  if (boxes && !map_rows(&tm_y, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.y, a.M, a.N, 2LL * a.N, 32)) return cudaErrorInvalidValue;
  const long long tiles = (long long)((a.M + 255) / 256) * ((a.N + P_BN - 1) / P_BN);
  cfg.gridDim = dim3((unsigned)(2 * (tiles < max_pairs ? tiles : max_pairs)));
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, gemm8_pair_kernel, tm_x, tm_w, tm_y, a, boxes);
}

// Clusters of `split` tiles' CTAs that are resident at once: one CTA fills an SM at every width.
int clusters_of(int split) {
  static const std::array<int, 9> counts = [] {
    std::array<int, 9> c{};
    c[1] = sm_count();
    if (cudaFuncSetAttribute(gemm8_tile_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileCfg<128>::SMEM) != cudaSuccess) return c;
    for (int s = 2; s <= 8; ++s) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(sm_count() / s * s));
      cfg.blockDim = dim3(kTileThreads);
      cfg.dynamicSmemBytes = TileCfg<128>::SMEM;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)s; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr; cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&c[s], gemm8_tile_kernel<128>, &cfg) != cudaSuccess) { (void)cudaGetLastError(); c[s] = 0; }
    }
    return c;
  }();
  return counts[split];
}

// Which kernel, tile and split: the shortest estimate in us. A wave of tiles costs its K blocks, more of them the more SMs take part (their
// copies share the L2), and every wave but the last the draining of its tiles; a split adds the exchange. The constants are fitted to
// 3157 launches of 256 products of 1 to 4096 rows, 256 to 4096 codes and 256 to 8192 outputs (replayed back to back); the chosen
// launches take 1.4 % more time in sum than the fastest of each product:
//   8 x 1024 x 8192 4.1 with 16 columns, 5.3 with 128; 8 x 4096 x 1000 4.4 split eight ways, 7.3 whole; 128 x 1024 x 8192 5.5 with 64 columns,
//   7.2 with 128, 7.5 on pairs; 1024 x 1024 x 8192 27.6 with 128 columns, 11.5 on pairs
void choose(const Gemm8Args& a, int* bn, int* split) {
  struct Cost { int bn; double base, block, load, wave, exchange; };
  static const Cost costs[5] = {{16, 2.85, 0.14, 0.03, 2.46, 0.96}, {32, 3.15, 0.13, 0.06, 2.85, 0.87}, {64, 3.49, 0.13, 0.12, 3.27, 0.80},
                                {128, 3.89, 0.13, 0.27, 3.73, 0.74}, {512, 5.02, 0.27, 0.09, 1.27, 0.0}};
  const long long num_kb = (a.K + KB - 1) / KB;
  double best = 1e30;
  for (const Cost& c : costs) {
    const bool pairs = c.bn == 512;
    const long long tiles = pairs ? (long long)((a.M + 255) / 256) * ((a.N + 255) / 256) : (long long)((a.M + c.bn - 1) / c.bn) * ((a.N + 127) / 128);
    for (int s = 1; s <= (pairs ? 1 : 8) && s <= num_kb; ++s) {
      const long long slots = pairs ? sm_count() / 2 : clusters_of(s);
      if (slots <= 0 || (s > 1 && tiles > slots)) continue;          // splitting more than what is resident at once only adds exchanges
      const double waves = (double)((tiles + slots - 1) / slots), blocks = waves * (double)((num_kb + s - 1) / s), load = tiles < slots ? (double)tiles / slots : 1.0;
      const double us = c.base + blocks * (c.block + c.load * load) + c.wave * (waves - 1) + (s > 1 ? c.exchange : 0.0);
      if (us < best) { best = us; *bn = c.bn; *split = s; }
    }
  }
}

}  // namespace

cudaError_t gemm_8bit(const Gemm8Args& a, int bn, int split, cudaStream_t st) {
  if (a.M <= 0 || a.N <= 0) return cudaSuccess;
  const int num_kb = (a.K + KB - 1) / KB;
  if (bn == 0) choose(a, &bn, &split);
  if (bn == 512) return launch_pairs(a, st);
  if (split == 0) split = 1;
  if (split < 1 || split > 8 || split > num_kb) return cudaErrorInvalidValue;
  switch (bn) {
    case 16: return launch_tiles<16>(a, split, st);
    case 32: return launch_tiles<32>(a, split, st);
    case 64: return launch_tiles<64>(a, split, st);
    case 128: return launch_tiles<128>(a, split, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace adb200
