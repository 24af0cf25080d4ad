// Gated linear recurrence over time, channel by channel:
//
//   h_t = f_t h_{t-1} + u_t x_t,   f = sigmoid(forget + bias),   u = sigmoid(input), or 1 - f without an input gate
//
// and f_t counts as 0 in front of h_{t-1} where `reset` says that the state is forgotten. Backward:
//
//   dh_t = dy_t + f_{t+1} dh_{t+1},   dx = dh u,   dforget = dh (h_{t-1} [- x]) f (1 - f),   dinput = dh x u (1 - u)
//
// Steps compose: a run of them takes h to A h + H, and two runs one after the other to (A2 A1) h + (A2 H1 + H2), so that pieces of a sequence
// are worked on at the same time and joined. A warp takes kSteps steps of 32 lanes' channels; its inputs are read once, 128 bytes a row, and
// stay in registers: it computes (A, H) of its steps, hears from the warps in front what state it starts from, and writes its outputs.
//
//   a thread block  is a tile of up to 8 warps' consecutive steps, joined through shared memory (or, for short sequences, several channel
//                   groups' tiles beside one another), and walks along its sequence tile by tile, the next tile's inputs on their way
//   a cluster       of S blocks takes S consecutive tiles at once where there are too few channels to fill the GPU: each block writes its
//                   (A, H) into the others' shared memory, one cluster barrier a round. Nothing spins on global memory and nothing
//                   is read twice; the order of joining is fixed.
//
// The states are not stored: the forward pass keeps them in fp32 in front of every tile, and the backward pass, which walks the other way with
// the same joining of dh, computes those in between again. States, gates and sums are fp32.
#include "recurrence.h"

#include <cuda_bf16.h>

#include "pair_tcgen05.cuh"
#include "pdl.cuh"
#include "sm_count.h"

namespace adb200 {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int kSteps = 8;                    // of a warp
constexpr int kWarps = 8;                    // of a block at most
constexpr int kMostSplit = 16;
static_assert(kSteps * kWarps == kScanTile, "a kept state in front of every tile");

// A lane's channels in one 32-bit word at most: two of bf16, or one.
template <typename T, int VEC> struct Lane;
template <> struct Lane<bf16, 2> {
  static __device__ __forceinline__ uint32_t load(const bf16* p) { return __ldg(reinterpret_cast<const uint32_t*>(p)); }
  static __device__ __forceinline__ void unpack(uint32_t w, float* v) { v[0] = __uint_as_float(w << 16); v[1] = __uint_as_float(w & 0xffff0000u); }
  static __device__ __forceinline__ void store(bf16* p, const float* v) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v[0], v[1]); }
};
template <> struct Lane<bf16, 1> {
  static __device__ __forceinline__ uint32_t load(const bf16* p) { return __ldg(reinterpret_cast<const unsigned short*>(p)); }
  static __device__ __forceinline__ void unpack(uint32_t w, float* v) { v[0] = __uint_as_float(w << 16); }
  static __device__ __forceinline__ void store(bf16* p, const float* v) { *p = __float2bfloat16(v[0]); }
};
template <> struct Lane<float, 1> {
  static __device__ __forceinline__ uint32_t load(const float* p) { return __ldg(reinterpret_cast<const uint32_t*>(p)); }
  static __device__ __forceinline__ void unpack(uint32_t w, float* v) { v[0] = __uint_as_float(w); }
  static __device__ __forceinline__ void store(float* p, const float* v) { *p = v[0]; }
};

// sigmoid(v) and 1 - sigmoid(v), neither of them by subtraction. For bf16 inputs with the approximate exponential and reciprocal, whose errors
// of a few 2^-23 are far below what the inputs were rounded by.
template <typename T> __device__ __forceinline__ float2 both_sides(float v);
template <> __device__ __forceinline__ float2 both_sides<float>(float v) {
  const float t = expf(-fabsf(v)), r = 1.0f / (1.0f + t);
  return v >= 0.f ? make_float2(r, t * r) : make_float2(t * r, r);
}
template <> __device__ __forceinline__ float2 both_sides<bf16>(float v) {
  const float t = __expf(-fabsf(v)), r = __fdividef(1.0f, 1.0f + t);
  const float s = t * r;
  return v >= 0.f ? make_float2(r, s) : make_float2(s, r);
}

// What steps do to a state: h -> A h + H. Decays are not negative; behind a forgotten state A is -0, and then nothing of h is left, not even
// an infinity.
__device__ __forceinline__ float after(float2 s, float h) { return __float_as_int(s.x) < 0 ? s.y : fmaf(s.x, h, s.y); }
__device__ __forceinline__ float2 joined(float2 first, float2 then) {
  const bool cut = __float_as_int(first.x) < 0 || __float_as_int(then.x) < 0;
  return make_float2(cut ? -0.0f : first.x * then.x, after(then, first.y));
}

__device__ __forceinline__ void store_cluster(uint32_t addr, float2 v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}

// Where a thread works. `warps`: warps of a tile; a block holds kWarps / warps tiles of neighbouring channel groups, or one.
template <int VEC>
struct Place {
  int lane, warp, part, first;               // part: the warp's place in its tile, whose first warp is `first`
  int b, c, rank;
  bool live;
  __device__ __forceinline__ Place(const ScanArgs& a, int warps, int split) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    part = warp % warps;
    first = warp - part;
    rank = split > 1 ? (int)tc::cluster_ctarank() : 0;
    const int across = (a.channels + 32 * VEC - 1) / (32 * VEC);
    const int column = blockIdx.x / split * (blockDim.x / 32 / warps) + warp / warps;
    b = column / across;
    c = column % across * 32 * VEC + lane * VEC;
    live = b < a.batch && c < a.channels;
  }
};

template <typename T> __device__ __forceinline__ const T* row_of(const ScanView& v, int b, int t, int c) { return static_cast<const T*>(v.p) + b * v.batch + t * v.step + c; }

template <typename T, int VEC, int N>
__device__ __forceinline__ void load_steps(uint32_t* raw, const ScanView& v, int b, int t0, int c, int steps, bool live) {
#pragma unroll
  for (int i = 0; i < N; ++i) raw[i] = live && t0 + i < steps ? Lane<T, VEC>::load(row_of<T>(v, b, t0 + i, c)) : 0u;
}
// Bit i: the state in front of step t0 + i is forgotten.
__device__ __forceinline__ uint32_t load_cuts(const ScanArgs& a, int b, int t0, int lane) {
  const bool cut = a.reset != nullptr && lane < kSteps && b < a.batch && t0 + lane < a.steps && a.reset[b * a.reset_batch + (long long)(t0 + lane) * a.reset_step] != 0;
  return __ballot_sync(0xffffffffu, cut);
}

template <typename T, int VEC, bool GATE>
__global__ void __launch_bounds__(32 * kWarps, 3)
scan_fwd_kernel(const ScanArgs a, T* __restrict__ y, float* __restrict__ last, float* __restrict__ kept, const int warps, const int split) {
  __shared__ float2 parts[2][kWarps][VEC][32];
  __shared__ float2 tiles[2][kMostSplit][VEC][32];
  pdl_sync();
  const Place<VEC> at(a, warps, split);
  const int tile_steps = warps * kSteps;
  const int count = (a.steps + tile_steps - 1) / tile_steps, rounds = (count + split - 1) / split;
  if (split > 1) tc::cluster_sync_all();       // the others' shared memory is there
  float carry[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) carry[v] = at.live && a.state != nullptr ? a.state[(long long)at.b * a.channels + at.c + v] : 0.f;

  uint32_t xr[kSteps], fr[kSteps], ir[GATE ? kSteps : 1], cuts;
  auto request = [&](int tile) {
    const int t0 = tile * tile_steps + at.part * kSteps;
    load_steps<T, VEC, kSteps>(fr, a.forget, at.b, t0, at.c, a.steps, at.live);
    load_steps<T, VEC, kSteps>(xr, a.x, at.b, t0, at.c, a.steps, at.live);
    if (GATE) load_steps<T, VEC, GATE ? kSteps : 1>(ir, a.input, at.b, t0, at.c, a.steps, at.live);
    cuts = load_cuts(a, at.b, t0, at.lane);
  };
  if (rounds > 0) request(at.rank);
  for (int k = 0; k < rounds; ++k) {
    const int tile = k * split + at.rank, t0 = tile * tile_steps + at.part * kSteps, buf = k & 1;
    float2 upto[kSteps][VEC];                  // what the steps up to each do to the state that this warp starts from
    float2 sum[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) sum[v] = make_float2(1.f, 0.f);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float x[VEC], g[VEC], in[VEC];
      Lane<T, VEC>::unpack(xr[i], x);
      Lane<T, VEC>::unpack(fr[i], g);
      if (GATE) Lane<T, VEC>::unpack(ir[GATE ? i : 0], in);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float2 f = both_sides<T>(g[v] + a.forget_bias);
        const float w = (GATE ? both_sides<T>(in[v]).x : f.y) * x[v];
        if (t0 + i < a.steps) sum[v] = cuts >> i & 1 ? make_float2(-0.0f, w) : make_float2(sum[v].x * f.x, fmaf(f.x, sum[v].y, w));
        upto[i][v] = sum[v];
      }
    }
    if (k + 1 < rounds) request(tile + split);
    float start[VEC];
    if (warps > 1 || split > 1) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) parts[buf][at.warp][v][at.lane] = sum[v];
      __syncthreads();
    }
    if (split > 1) {
      // the tile as a whole, to every block of the cluster
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float2 whole = parts[buf][0][v][at.lane];
        for (int j = 1; j < warps; ++j) whole = joined(whole, parts[buf][j][v][at.lane]);
        for (int r = at.warp; r < split; r += kWarps) store_cluster(tc::map_to_cta(tc::smem_u32(&tiles[buf][at.rank][v][at.lane]), (uint32_t)r), whole);
      }
      __syncwarp();
      tc::cluster_sync_all();
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float h = carry[v];
      if (split > 1) {
        float front = h;
        for (int r = 0; r < split; ++r) {
          if (r == at.rank) front = h;
          h = after(tiles[buf][r][v][at.lane], h);
        }
        carry[v] = h;
        h = front;
      }
      start[v] = h;
      if (kept != nullptr && at.part == 0 && at.live && tile < count) kept[((long long)at.b * count + tile) * a.channels + at.c + v] = h;
      if (warps > 1) {
        for (int j = 0; j < warps; ++j) {
          if (j == at.part) start[v] = h;
          h = after(parts[buf][at.first + j][v][at.lane], h);
        }
      } else {
        h = after(sum[v], h);
      }
      if (split == 1) carry[v] = h;
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (at.live && t0 + i < a.steps) {
        float h[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = after(upto[i][v], start[v]);
        Lane<T, VEC>::store(y + ((long long)at.b * a.steps + t0 + i) * a.channels + at.c, h);
      }
    }
  }
  if (at.rank == 0 && at.part == 0 && at.live) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) last[(long long)at.b * a.channels + at.c + v] = carry[v];
  }
}

template <typename T, int VEC, bool GATE>
__global__ void __launch_bounds__(32 * kWarps, 2)
scan_bwd_kernel(const ScanArgs a, const ScanGrads g, const int warps, const int split) {
  __shared__ float2 parts[2][kWarps][VEC][32];           // (A, H) of a warp's steps
  __shared__ float back[2][kWarps][VEC][32];             // their dh: from the end of the steps to their front it is A dh + back
  __shared__ float2 tiles[2][kMostSplit][VEC][32];       // (A, back) of a tile
  pdl_sync();
  const Place<VEC> at(a, warps, split);
  const int tile_steps = warps * kSteps;
  const int count = (a.steps + tile_steps - 1) / tile_steps, rounds = (count + split - 1) / split;
  if (split > 1) tc::cluster_sync_all();
  float carry[VEC];                                      // f_{t+1} dh_{t+1} at the end of what is left
#pragma unroll
  for (int v = 0; v < VEC; ++v) carry[v] = at.live && g.dlast != nullptr ? g.dlast[(long long)at.b * a.channels + at.c + v] : 0.f;

  uint32_t xr[kSteps], fr[kSteps], ir[GATE ? kSteps : 1], dr[kSteps], cuts;
  float front[VEC];
  auto request = [&](int tile) {
    const int t0 = tile * tile_steps + at.part * kSteps;
    load_steps<T, VEC, kSteps>(fr, a.forget, at.b, t0, at.c, a.steps, at.live);
    load_steps<T, VEC, kSteps>(xr, a.x, at.b, t0, at.c, a.steps, at.live);
    if (GATE) load_steps<T, VEC, GATE ? kSteps : 1>(ir, a.input, at.b, t0, at.c, a.steps, at.live);
    load_steps<T, VEC, kSteps>(dr, g.dy, at.b, t0, at.c, a.steps, at.live && g.dy.p != nullptr);
    cuts = load_cuts(a, at.b, t0, at.lane);
#pragma unroll
    for (int v = 0; v < VEC; ++v) front[v] = at.live && tile < count ? g.kept[((long long)at.b * count + tile) * a.channels + at.c + v] : 0.f;
  };
  if (rounds > 0) request((rounds - 1) * split + at.rank);
  for (int k = rounds - 1; k >= 0; --k) {
    const int tile = k * split + at.rank, t0 = tile * tile_steps + at.part * kSteps, buf = k & 1;
    float f[kSteps][VEC], n[kSteps][VEC];                // sigmoid and its complement
    float u[GATE ? kSteps : 1][VEC], m[GATE ? kSteps : 1][VEC];
    float2 sum[VEC];
    float up[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { sum[v] = make_float2(1.f, 0.f); up[v] = 0.f; }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float x[VEC], w[VEC], in[VEC];
      Lane<T, VEC>::unpack(xr[i], x);
      Lane<T, VEC>::unpack(fr[i], w);
      if (GATE) Lane<T, VEC>::unpack(ir[GATE ? i : 0], in);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float2 s = both_sides<T>(w[v] + a.forget_bias);
        f[i][v] = s.x;
        n[i][v] = s.y;
        if (GATE) {
          const float2 t = both_sides<T>(in[v]);
          u[GATE ? i : 0][v] = t.x;
          m[GATE ? i : 0][v] = t.y;
        }
        const float add = (GATE ? u[GATE ? i : 0][v] : s.y) * x[v];
        if (t0 + i < a.steps) sum[v] = cuts >> i & 1 ? make_float2(-0.0f, add) : make_float2(sum[v].x * s.x, fmaf(s.x, sum[v].y, add));
      }
    }
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      float dy[VEC];
      Lane<T, VEC>::unpack(dr[i], dy);
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (t0 + i < a.steps) up[v] = cuts >> i & 1 ? 0.f : f[i][v] * (dy[v] + up[v]);
    }
    float start[VEC], end[VEC];
    if (warps > 1 || split > 1) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        parts[buf][at.warp][v][at.lane] = sum[v];
        back[buf][at.warp][v][at.lane] = up[v];
      }
      __syncthreads();
    }
    if (split > 1) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float2 whole = make_float2(1.f, 0.f);
        for (int j = warps - 1; j >= 0; --j) whole = joined(whole, make_float2(parts[buf][j][v][at.lane].x, back[buf][j][v][at.lane]));
        for (int r = at.warp; r < split; r += kWarps) store_cluster(tc::map_to_cta(tc::smem_u32(&tiles[buf][at.rank][v][at.lane]), (uint32_t)r), whole);
      }
      __syncwarp();
      tc::cluster_sync_all();
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float d = carry[v];
      if (split > 1) {
        float behind = d;
        for (int r = split - 1; r >= 0; --r) {
          if (r == at.rank) behind = d;
          d = after(tiles[buf][r][v][at.lane], d);
        }
        carry[v] = d;
        d = behind;
      }
      end[v] = d;
      start[v] = front[v];
      if (warps > 1) {
        float h = front[v];
        for (int j = 0; j < at.part; ++j) h = after(parts[buf][at.first + j][v][at.lane], h);
        start[v] = h;
        for (int j = warps - 1; j >= 0; --j) {
          if (j == at.part) end[v] = d;
          d = after(make_float2(parts[buf][at.first + j][v][at.lane].x, back[buf][at.first + j][v][at.lane]), d);
        }
      } else {
        d = after(make_float2(sum[v].x, up[v]), d);
      }
      if (split == 1) carry[v] = d;
    }
    // the states in front of each step, then dh from the last step to the first
    float before[kSteps][VEC];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float x[VEC];
      Lane<T, VEC>::unpack(xr[i], x);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        before[i][v] = cuts >> i & 1 ? 0.f : start[v];
        start[v] = fmaf(f[i][v], before[i][v], (GATE ? u[GATE ? i : 0][v] : n[i][v]) * x[v]);
      }
    }
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      if (t0 + i < a.steps) {
        float x[VEC], dy[VEC], dx[VEC], df[VEC], di[VEC];
        Lane<T, VEC>::unpack(xr[i], x);
        Lane<T, VEC>::unpack(dr[i], dy);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float dh = end[v] + dy[v];
          dx[v] = dh * (GATE ? u[GATE ? i : 0][v] : n[i][v]);
          df[v] = dh * (GATE ? before[i][v] : before[i][v] - x[v]) * (f[i][v] * n[i][v]);
          if (GATE) di[v] = dh * x[v] * (u[GATE ? i : 0][v] * m[GATE ? i : 0][v]);
          end[v] = cuts >> i & 1 ? 0.f : f[i][v] * dh;
        }
        if (at.live) {
          const long long out = ((long long)at.b * a.steps + t0 + i) * a.channels + at.c;
          Lane<T, VEC>::store(static_cast<T*>(g.dx) + out, dx);
          Lane<T, VEC>::store(static_cast<T*>(g.dforget) + out, df);
          if (GATE) Lane<T, VEC>::store(static_cast<T*>(g.dinput) + out, di);
        }
      }
    }
    if (k > 0) request(tile - split);
  }
  if (at.rank == 0 && at.part == 0 && at.live) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) g.dstate[(long long)at.b * a.channels + at.c + v] = carry[v];
  }
}

struct Shape { int warps, split, threads; unsigned blocks; };
// How a call is laid out: as many warps a tile as the sequence fills, several tiles of short sequences in a block, and a cluster along time
// where the channels alone do not fill the SMs.
Shape shape_of(const ScanArgs& a, int vec) {
  const long long columns = (long long)a.batch * ((a.channels + 32 * vec - 1) / (32 * vec));
  Shape s;
  s.warps = (a.steps + kSteps - 1) / kSteps;
  s.warps = s.warps < 1 ? 1 : s.warps > kWarps ? kWarps : s.warps;
  const int beside = kWarps / s.warps;
  s.threads = 32 * s.warps * beside;
  s.split = 1;
  const long long tiles = (a.steps + kScanTile - 1) / kScanTile;
  while (s.split < kMostSplit && tiles >= 2 * s.split && columns * s.split < 3LL * sm_count()) s.split *= 2;
  s.blocks = (unsigned)((columns + beside - 1) / beside * s.split);
  return s;
}

template <typename... K, typename... A>
cudaError_t launch(void (*kernel)(K...), const Shape& s, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.blocks);
  cfg.blockDim = dim3(s.threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)s.split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = s.split > 1 ? 2 : 1;
  if (s.split > 8) {                         // clusters of more than 8 blocks have to be asked for
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args..., s.warps, s.split);
}

bool pairs_fit(const ScanView& v) { return reinterpret_cast<uintptr_t>(v.p) % 4 == 0 && v.batch % 2 == 0 && v.step % 2 == 0; }

template <typename T, int VEC>
cudaError_t forward(const ScanArgs& a, void* y, float* last, float* kept, cudaStream_t st) {
  const Shape s = shape_of(a, VEC);
  return a.input.p != nullptr ? launch(scan_fwd_kernel<T, VEC, true>, s, st, a, static_cast<T*>(y), last, kept)
                              : launch(scan_fwd_kernel<T, VEC, false>, s, st, a, static_cast<T*>(y), last, kept);
}
template <typename T, int VEC>
cudaError_t backward(const ScanArgs& a, const ScanGrads& g, cudaStream_t st) {
  const Shape s = shape_of(a, VEC);
  return a.input.p != nullptr ? launch(scan_bwd_kernel<T, VEC, true>, s, st, a, g) : launch(scan_bwd_kernel<T, VEC, false>, s, st, a, g);
}
bool in_pairs(const ScanArgs& a) { return a.channels % 2 == 0 && pairs_fit(a.x) && pairs_fit(a.forget) && (a.input.p == nullptr || pairs_fit(a.input)); }

}  // namespace

cudaError_t gated_scan_fwd(const ScanArgs& a, void* y, float* last, float* kept, cudaStream_t st) {
  if (a.batch <= 0 || a.channels <= 0) return cudaSuccess;
  if (!a.bf16) return forward<float, 1>(a, y, last, kept, st);
  return in_pairs(a) ? forward<bf16, 2>(a, y, last, kept, st) : forward<bf16, 1>(a, y, last, kept, st);
}
cudaError_t gated_scan_bwd(const ScanArgs& a, const ScanGrads& g, cudaStream_t st) {
  if (a.batch <= 0 || a.channels <= 0) return cudaSuccess;
  if (!a.bf16) return backward<float, 1>(a, g, st);
  return in_pairs(a) && (g.dy.p == nullptr || pairs_fit(g.dy)) ? backward<bf16, 2>(a, g, st) : backward<bf16, 1>(a, g, st);
}

}  // namespace adb200
