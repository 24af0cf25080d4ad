// Gated linear recurrence over time, channel by channel:
//
//   h_t = f_t h_{t-1} + u_t x_t,   f = sigmoid(forget + bias),   u = sigmoid(input), or 1 - f without an input gate
//
// and f_t counts as 0 in front of h_{t-1} where `reset` says that the state is forgotten. Backward:
//
//   dh_t = dy_t + f_{t+1} dh_{t+1},   dx = dh u,   dforget = dh (h_{t-1} [- x]) f (1 - f),   dinput = dh x u (1 - u)
//
// Steps compose: a run of them takes h to A h + H, and two runs one after the other to (A2 A1) h + (A2 H1 + H2), so that pieces of a sequence
// are worked on at the same time and joined. A warp takes 8 or 16 steps of 32 lanes' channels: it computes (A, H) of its steps with the gates
// left in registers, hears what state it starts from, and walks through them. Every input is read once.
//
//   a warp          walks along its sequence alone where there are enough of them; its inputs come ahead of it into a ring of its own in
//                   shared memory (cp.async), so that a wait of one warp holds up no other
//   a thread block  of up to 8 warps takes as many runs of steps side by side, joined through shared memory, where there are fewer channels
//   a cluster       of S blocks takes S such tiles at once where there are fewer still: each block writes its (A, H) into the others'
//                   shared memory, one cluster barrier a round. Nothing spins on global memory; the order of joining is fixed.
//
// The states are not stored: the forward pass keeps them in fp32 in front of every tile of the backward pass, which walks the other way with
// the same joining of dh and computes those in between again. States, gates and sums are fp32.
#include "recurrence.h"

#include <cuda_bf16.h>

#include <initializer_list>

#include "pair_tcgen05.cuh"
#include "pdl.cuh"
#include "sm_count.h"

namespace adb200 {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int kWarps = 8;                    // of a block at most
constexpr int kBack = 8;                     // steps of a warp in the backward pass
constexpr int kMostSplit = 16;

// fp32 values of a lane's channels, one or two of them; two take one instruction.
template <int VEC> struct F;
template <> struct F<1> { float v; };
template <> struct F<2> { uint64_t v; };
__device__ __forceinline__ F<1> add(F<1> a, F<1> b) { return {a.v + b.v}; }
__device__ __forceinline__ F<1> mul(F<1> a, F<1> b) { return {a.v * b.v}; }
__device__ __forceinline__ F<1> fma(F<1> a, F<1> b, F<1> c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ F<2> add(F<2> a, F<2> b) { return {tc::add2(a.v, b.v)}; }
__device__ __forceinline__ F<2> mul(F<2> a, F<2> b) { return {tc::mul2(a.v, b.v)}; }
__device__ __forceinline__ F<2> fma(F<2> a, F<2> b, F<2> c) { return {tc::fma2(a.v, b.v, c.v)}; }
template <int VEC> __device__ __forceinline__ F<VEC> all(float x);
template <> __device__ __forceinline__ F<1> all<1>(float x) { return {x}; }
template <> __device__ __forceinline__ F<2> all<2>(float x) { return {tc::pack_f32x2(x, x)}; }
template <class Fn> __device__ __forceinline__ F<1> each(F<1> a, Fn fn) { return {fn(a.v)}; }
template <class Fn> __device__ __forceinline__ F<2> each(F<2> a, Fn fn) {
  const float2 x = tc::unpack_f32x2(a.v);
  return {tc::pack_f32x2(fn(x.x), fn(x.y))};
}
// `then` in channels where the sign of `a` is set, else `other`
__device__ __forceinline__ F<1> where_cut(F<1> a, F<1> then, F<1> other) { return {__float_as_int(a.v) < 0 ? then.v : other.v}; }
__device__ __forceinline__ F<2> where_cut(F<2> a, F<2> then, F<2> other) {
  const float2 x = tc::unpack_f32x2(a.v), t = tc::unpack_f32x2(then.v), o = tc::unpack_f32x2(other.v);
  return {tc::pack_f32x2(__float_as_int(x.x) < 0 ? t.x : o.x, __float_as_int(x.y) < 0 ? t.y : o.y)};
}
__device__ __forceinline__ F<1> load_f(const float* p, F<1>*) { return {*p}; }
__device__ __forceinline__ F<2> load_f(const float* p, F<2>*) {
  const float2 x = *reinterpret_cast<const float2*>(p);
  return {tc::pack_f32x2(x.x, x.y)};
}
__device__ __forceinline__ void store_f(float* p, F<1> a) { *p = a.v; }
__device__ __forceinline__ void store_f(float* p, F<2> a) { *reinterpret_cast<float2*>(p) = tc::unpack_f32x2(a.v); }

// A lane's channels as they lie in memory. kOpen: forget gates that are open, for steps that are not there.
template <typename T, int VEC> struct Lane;
template <> struct Lane<bf16, 2> {
  typedef uint32_t Raw;
  static constexpr Raw kOpen = 0x7F807F80u;
  static __device__ __forceinline__ F<2> unpack(Raw w) { return {tc::widen2(w)}; }
  static __device__ __forceinline__ void store(bf16* p, F<2> a) { *reinterpret_cast<uint32_t*>(p) = tc::round2(a.v); }
};
template <> struct Lane<bf16, 1> {
  typedef unsigned short Raw;
  static constexpr Raw kOpen = 0x7F80u;
  static __device__ __forceinline__ F<1> unpack(Raw w) { return {__uint_as_float((uint32_t)w << 16)}; }
  static __device__ __forceinline__ void store(bf16* p, F<1> a) { *p = __float2bfloat16(a.v); }
};
template <> struct Lane<float, 1> {
  typedef uint32_t Raw;
  static constexpr Raw kOpen = 0x7F800000u;
  static __device__ __forceinline__ F<1> unpack(Raw w) { return {__uint_as_float(w)}; }
  static __device__ __forceinline__ void store(float* p, F<1> a) { *p = a.v; }
};
template <> struct Lane<float, 2> {
  typedef uint64_t Raw;
  static constexpr Raw kOpen = 0x7F8000007F800000ull;
  static __device__ __forceinline__ F<2> unpack(Raw w) { return {w}; }
  static __device__ __forceinline__ void store(float* p, F<2> a) { store_f(p, a); }
};

__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp_fast(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

constexpr float kLog2e = 1.4426950408889634f;

// sigmoid(g + bias) = 1 / (1 + e) and its complement e / (1 + e), neither by subtraction, with e = 2^(-(g + bias) log2(e)). e is kept
// finite: a gate shut by minus infinity still lets some 2^-126 through.
//   bf16  the exponent in one rounding: e is off by |g| 2^-24 or so, far below what the rounding of g to 8 bits did to it
//   fp32  what the product with log2(e) cut off is put back, so that e is off by the exponential's own two last bits
template <typename T, int VEC> struct Gate;
template <int VEC> struct Gate<bf16, VEC> {
  F<VEC> bias;
  __device__ __forceinline__ explicit Gate(float b) : bias(all<VEC>(-kLog2e * b)) {}
  __device__ __forceinline__ void operator()(F<VEC> g, F<VEC>& f, F<VEC>& n) const {
    const F<VEC> e = each(fma(g, all<VEC>(-kLog2e), bias), [](float x) { return exp2_fast(min_nan(x, 126.f)); });
    f = each(add(e, all<VEC>(1.f)), rcp_fast);
    n = mul(e, f);
  }
};
template <int VEC> struct Gate<float, VEC> {
  F<VEC> bias;
  __device__ __forceinline__ explicit Gate(float b) : bias(all<VEC>(b)) {}
  __device__ __forceinline__ void operator()(F<VEC> g, F<VEC>& f, F<VEC>& n) const {
    const F<VEC> z = each(add(g, bias), [](float x) { return min_nan(max_nan(x, -87.f), 110.f); });
    const F<VEC> x = mul(z, all<VEC>(-kLog2e));
    const F<VEC> cut = fma(z, all<VEC>(-1.925963033500e-08f), fma(z, all<VEC>(-kLog2e), mul(x, all<VEC>(-1.f))));     // log2(e) is kLog2e + 1.926e-8
    const F<VEC> p = each(x, exp2_fast);
    const F<VEC> e = fma(p, mul(cut, all<VEC>(0.69314718f)), p);
    f = each(add(e, all<VEC>(1.f)), rcp_fast);
    n = mul(e, f);
  }
};

// What steps do to a state: h -> a h + b. Decays are not negative; CUT: behind a forgotten state a is -0, and then nothing of h is left, not
// even an infinity.
template <int VEC> struct Run { F<VEC> a, b; };
template <bool CUT, int VEC> __device__ __forceinline__ F<VEC> after(const Run<VEC>& s, F<VEC> h) {
  const F<VEC> r = fma(s.a, h, s.b);
  return CUT ? where_cut(s.a, s.b, r) : r;
}
template <bool CUT, int VEC> __device__ __forceinline__ Run<VEC> joined(const Run<VEC>& first, const Run<VEC>& then) {
  F<VEC> a = mul(first.a, then.a);
  if (CUT) a = where_cut(first.a, all<VEC>(-0.f), where_cut(then.a, all<VEC>(-0.f), a));
  return {a, after<CUT>(then, first.b)};
}

__device__ __forceinline__ void store_cluster(uint32_t addr, Run<1> r) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(r.a.v), "f"(r.b.v) : "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, Run<2> r) {
  asm volatile("st.shared::cluster.v2.b64 [%0], {%1, %2};" ::"r"(addr), "l"(r.a.v), "l"(r.b.v) : "memory");
}

// Where a thread works. `warps`: warps of a tile; a block holds kWarps / warps tiles of neighbouring channel groups, or one.
template <int VEC>
struct Place {
  int lane, warp, part, first;               // part: the warp's place in its tile, whose first warp is `first`
  int b, c0, c, rank;                        // c0: the warp's first channel
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
    c0 = column % across * 32 * VEC;
    c = c0 + lane * VEC;
    live = b < a.batch && c < a.channels;
  }
};

template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// How a warp's ring of inputs lies in shared memory: `SLOTS` tiles of NT tensors' STEPS rows.
template <typename T, int VEC, int STEPS, int NT>
struct Ring {
  typedef typename Lane<T, VEC>::Raw Raw;
  static constexpr int ROW = 32 * VEC * (int)sizeof(T);
  static constexpr int SLOT = NT * STEPS * ROW;
  static constexpr int FIT = 84 * 1024 / (kWarps * SLOT);       // two blocks and what they exchange through on an SM
  static constexpr int SLOTS = FIT < 2 ? 2 : FIT > 4 ? 4 : FIT;
  static constexpr int BYTES = SLOTS * SLOT;             // of a warp
};

// Requests one tensor's rows t0 ... of a warp's channels; rows and channels that are not there hold `none`. `wide`: whole 16-byte pieces.
template <typename T, int VEC, int STEPS>
__device__ __forceinline__ void request_rows(uint8_t* dst, const ScanView& v, int b, int t0, int rows, int c0, int channels, int lane, bool wide,
                                             typename Lane<T, VEC>::Raw none) {
  typedef typename Lane<T, VEC>::Raw Raw;
  constexpr int ROW = 32 * VEC * (int)sizeof(T), PIECES = ROW / 16, PER = 32 / PIECES;
  const T* base = static_cast<const T*>(v.p) + b * v.batch + t0 * v.step + c0;
  if (wide) {
    const int piece = lane % PIECES, c = piece * (16 / (int)sizeof(T));
    const T* src = base + lane / PIECES * v.step + c;
    uint8_t* to = dst + lane * 16;
    const int left = c0 + c < channels ? rows - lane / PIECES : 0;
#pragma unroll
    for (int i = 0; i < (STEPS + PER - 1) / PER; ++i, src += PER * v.step, to += 512) {
      if (STEPS % PER != 0 && i * PER + lane / PIECES >= STEPS) break;
      if (i * PER < left) {
        copy_async<16>(tc::smem_u32(to), src);
      } else {
#pragma unroll
        for (int j = 0; j < 16 / (int)sizeof(Raw); ++j) reinterpret_cast<Raw*>(to)[j] = none;
      }
    }
  } else {
    const T* src = base + lane * VEC;
    Raw* to = reinterpret_cast<Raw*>(dst) + lane;
    const int left = c0 + lane * VEC < channels ? rows : 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i, src += v.step, to += 32) {
      if (i < left) {
        if constexpr (sizeof(Raw) >= 4) copy_async<sizeof(Raw)>(tc::smem_u32(to), src);
        else *to = *reinterpret_cast<const Raw*>(src);
      } else {
        *to = none;
      }
    }
  }
}
// Bit i: the state in front of step t0 + i is forgotten.
template <int STEPS>
__device__ __forceinline__ uint32_t load_cuts(const ScanArgs& a, int b, int t0, int lane) {
  const bool cut = lane < STEPS && b < a.batch && t0 >= 0 && t0 + lane < a.steps && a.reset[b * a.reset_batch + (long long)(t0 + lane) * a.reset_step] != 0;
  return __ballot_sync(0xffffffffu, cut);
}

template <typename T, int VEC, bool GATE, bool CUT, int STEPS>
__global__ void __launch_bounds__(32 * kWarps, 2)
scan_fwd_kernel(const ScanArgs a, T* __restrict__ y, float* __restrict__ last, float* __restrict__ kept, const int keep, const int wide, const int warps,
                const int split) {
  typedef Lane<T, VEC> L;
  typedef F<VEC> V;
  typedef Ring<T, VEC, STEPS, GATE ? 3 : 2> R;
  extern __shared__ __align__(16) uint8_t ring_all[];
  __shared__ Run<VEC> parts[2][kWarps][32];
  __shared__ Run<VEC> tiles[2][kMostSplit][32];
  pdl_sync();
  const Place<VEC> at(a, warps, split);
  const int tile_steps = warps * STEPS;
  const int count = (a.steps + tile_steps - 1) / tile_steps, rounds = (count + split - 1) / split;
  uint8_t* ring = ring_all + at.warp * R::BYTES;
  const bool there = at.b < a.batch;
  auto request = [&](int k) {
    const int t0 = (k * split + at.rank) * tile_steps + at.part * STEPS;
    if (k < rounds) {
      uint8_t* slot = ring + k % R::SLOTS * R::SLOT;
      const int rows = there ? a.steps - t0 : 0;
      request_rows<T, VEC, STEPS>(slot, a.forget, at.b, t0, rows, at.c0, a.channels, at.lane, wide, L::kOpen);
      request_rows<T, VEC, STEPS>(slot + STEPS * R::ROW, a.x, at.b, t0, rows, at.c0, a.channels, at.lane, wide, 0);
      if constexpr (GATE) request_rows<T, VEC, STEPS>(slot + 2 * STEPS * R::ROW, a.input, at.b, t0, rows, at.c0, a.channels, at.lane, wide, 0);
    }
    commit_copies();
  };
#pragma unroll
  for (int k = 0; k < R::SLOTS - 1; ++k) request(k);
  const long long state_at = (long long)at.b * a.channels + at.c;
  V carry = at.live && a.state != nullptr ? load_f(a.state + state_at, static_cast<V*>(nullptr)) : all<VEC>(0.f);
  const Gate<T, VEC> forget(a.forget_bias), input(0.f);
  uint32_t cuts = 0, next_cuts = 0;
  if (CUT) next_cuts = load_cuts<STEPS>(a, at.b, at.rank * tile_steps + at.part * STEPS, at.lane);
  if (split > 1) tc::cluster_sync_all();       // the others' shared memory is there

  for (int k = 0; k < rounds; ++k) {
    const int tile = k * split + at.rank, t0 = tile * tile_steps + at.part * STEPS, buf = k & 1;
    request(k + R::SLOTS - 1);
    wait_copies<R::SLOTS - 1>();
    __syncwarp();
    if (CUT) {
      cuts = next_cuts;
      if (k + 1 < rounds) next_cuts = load_cuts<STEPS>(a, at.b, t0 + split * tile_steps, at.lane);
    }
    const typename L::Raw* raw = reinterpret_cast<const typename L::Raw*>(ring + k % R::SLOTS * R::SLOT) + at.lane;
    V f[STEPS], w[STEPS];
    Run<VEC> sum = {all<VEC>(1.f), all<VEC>(0.f)};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      V n;
      forget(L::unpack(raw[i * 32]), f[i], n);
      if constexpr (GATE) {
        V m;
        input(L::unpack(raw[(2 * STEPS + i) * 32]), n, m);
      }
      w[i] = mul(n, L::unpack(raw[(STEPS + i) * 32]));
      if (i == 0) sum = {f[0], w[0]};
      else sum = {mul(sum.a, f[i]), fma(f[i], sum.b, w[i])};
      if (CUT && (cuts >> i & 1)) sum = {all<VEC>(-0.f), w[i]};
    }
    __syncwarp();                              // the slot has been read
    if (warps > 1) {
      parts[buf][at.warp][at.lane] = sum;
      __syncthreads();
    }
    V h = carry;
    if (split > 1) {
      // the tile as a whole, to every block of the cluster
      Run<VEC> whole = parts[buf][0][at.lane];
#pragma unroll
      for (int j = 1; j < kWarps; ++j) whole = joined<CUT>(whole, parts[buf][j][at.lane]);
      for (int r = at.warp; r < split; r += kWarps) store_cluster(tc::map_to_cta(tc::smem_u32(&tiles[buf][at.rank][at.lane]), (uint32_t)r), whole);
      __syncwarp();
      tc::cluster_sync_all();
      V front = h;
#pragma unroll 4
      for (int r = 0; r < split; ++r) {
        if (r == at.rank) front = h;
        h = after<CUT>(tiles[buf][r][at.lane], h);
      }
      carry = h;
      h = front;
    }
    V start = h;
    if (warps == kWarps) {
#pragma unroll
      for (int j = 0; j < kWarps; ++j) {
        if (j == at.part) start = h;
        h = after<CUT>(parts[buf][j][at.lane], h);
      }
    } else if (warps > 1) {
      for (int j = 0; j < warps; ++j) {
        if (j == at.part) start = h;
        h = after<CUT>(parts[buf][at.first + j][at.lane], h);
      }
    } else {
      h = after<CUT>(sum, h);
    }
    if (split == 1) carry = h;
    const int rows = at.live ? a.steps - t0 : 0;
    // states in front of the backward pass's tiles, whose length is a multiple of this warp's steps, or half of them
    if (kept != nullptr && rows > 0) {
      if (t0 % keep == 0) store_f(kept + ((long long)at.b * ((a.steps + keep - 1) / keep) + t0 / keep) * a.channels + at.c, start);
    }
    T* out = y + ((long long)at.b * a.steps + t0) * a.channels + at.c;
    h = start;
#pragma unroll
    for (int i = 0; i < STEPS; ++i, out += a.channels) {
      if (STEPS > kBack && i == kBack && kept != nullptr && keep == kBack && i < rows)
        store_f(kept + ((long long)at.b * ((a.steps + keep - 1) / keep) + (t0 + i) / keep) * a.channels + at.c, h);
      h = CUT && (cuts >> i & 1) ? w[i] : fma(f[i], h, w[i]);
      if (i < rows) L::store(out, h);
    }
  }
  wait_copies<0>();
  if (at.rank == 0 && at.part == 0 && at.live) store_f(last + state_at, carry);
}

template <typename T, int VEC, bool GATE, bool CUT>
__global__ void __launch_bounds__(32 * kWarps, 2)
scan_bwd_kernel(const ScanArgs a, const ScanGrads g, const int wide, const int warps, const int split) {
  typedef Lane<T, VEC> L;
  typedef F<VEC> V;
  constexpr int STEPS = kBack;
  typedef Ring<T, VEC, STEPS, GATE ? 4 : 3> R;
  extern __shared__ __align__(16) uint8_t ring_all[];
  __shared__ Run<VEC> parts[2][kWarps][32];              // of a warp's steps
  __shared__ V back[2][kWarps][32];                      // their dh: from the end of the steps to their front it is a dh + back
  __shared__ Run<VEC> tiles[2][kMostSplit][32];          // a and back of a tile
  pdl_sync();
  const Place<VEC> at(a, warps, split);
  const int tile_steps = warps * STEPS;
  const int count = (a.steps + tile_steps - 1) / tile_steps, rounds = (count + split - 1) / split;
  uint8_t* ring = ring_all + at.warp * R::BYTES;
  const bool there = at.b < a.batch;
  // rounds are counted from the last tiles to the first
  auto t0_of = [&](int k) { return ((rounds - 1 - k) * split + at.rank) * tile_steps + at.part * STEPS; };
  auto request = [&](int k) {
    if (k < rounds) {
      const int t0 = t0_of(k), rows = there ? a.steps - t0 : 0;
      uint8_t* slot = ring + k % R::SLOTS * R::SLOT;
      request_rows<T, VEC, STEPS>(slot, a.forget, at.b, t0, rows, at.c0, a.channels, at.lane, wide, L::kOpen);
      request_rows<T, VEC, STEPS>(slot + STEPS * R::ROW, a.x, at.b, t0, rows, at.c0, a.channels, at.lane, wide, 0);
      request_rows<T, VEC, STEPS>(slot + 2 * STEPS * R::ROW, g.dy, at.b, t0, g.dy.p != nullptr ? rows : 0, at.c0, a.channels, at.lane, wide, 0);
      if constexpr (GATE) request_rows<T, VEC, STEPS>(slot + 3 * STEPS * R::ROW, a.input, at.b, t0, rows, at.c0, a.channels, at.lane, wide, 0);
    }
    commit_copies();
  };
  auto front_of = [&](int k) {
    const int tile = (rounds - 1 - k) * split + at.rank;
    return at.live && k < rounds && tile < count ? load_f(g.kept + ((long long)at.b * count + tile) * a.channels + at.c, static_cast<V*>(nullptr)) : all<VEC>(0.f);
  };
#pragma unroll
  for (int k = 0; k < R::SLOTS - 1; ++k) request(k);
  const long long state_at = (long long)at.b * a.channels + at.c;
  // f_{t+1} dh_{t+1} at the end of what is left
  V carry = at.live && g.dlast != nullptr ? load_f(g.dlast + state_at, static_cast<V*>(nullptr)) : all<VEC>(0.f);
  V next_front = front_of(0);
  const Gate<T, VEC> forget(a.forget_bias), input(0.f);
  uint32_t cuts = 0, next_cuts = 0;
  if (CUT) next_cuts = load_cuts<STEPS>(a, at.b, t0_of(0), at.lane);
  if (split > 1) tc::cluster_sync_all();

  for (int k = 0; k < rounds; ++k) {
    const int t0 = t0_of(k), buf = k & 1;
    request(k + R::SLOTS - 1);
    wait_copies<R::SLOTS - 1>();
    __syncwarp();
    V start = next_front;
    next_front = front_of(k + 1);
    if (CUT) {
      cuts = next_cuts;
      if (k + 1 < rounds) next_cuts = load_cuts<STEPS>(a, at.b, t0_of(k + 1), at.lane);
    }
    const typename L::Raw* raw = reinterpret_cast<const typename L::Raw*>(ring + k % R::SLOTS * R::SLOT) + at.lane;
    auto x_of = [&](int i) { return L::unpack(raw[(STEPS + i) * 32]); };
    auto dy_of = [&](int i) { return L::unpack(raw[(2 * STEPS + i) * 32]); };
    V f[STEPS], n[STEPS], u[GATE ? STEPS : 1], m[GATE ? STEPS : 1];              // sigmoids and their complements
    Run<VEC> sum = {all<VEC>(1.f), all<VEC>(0.f)};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      forget(L::unpack(raw[i * 32]), f[i], n[i]);
      if constexpr (GATE) input(L::unpack(raw[(3 * STEPS + i) * 32]), u[i], m[i]);
      const V w = mul(GATE ? u[GATE ? i : 0] : n[i], x_of(i));
      if (i == 0) sum = {f[0], w};
      else sum = {mul(sum.a, f[i]), fma(f[i], sum.b, w)};
      if (CUT && (cuts >> i & 1)) sum = {all<VEC>(-0.f), w};
    }
    V up = all<VEC>(0.f);
#pragma unroll
    for (int i = STEPS - 1; i >= 0; --i) {
      up = mul(f[i], add(dy_of(i), up));
      if (CUT && (cuts >> i & 1)) up = all<VEC>(0.f);
    }
    if (warps > 1) {
      parts[buf][at.warp][at.lane] = sum;
      back[buf][at.warp][at.lane] = up;
      __syncthreads();
    }
    V d = carry;
    if (split > 1) {
      Run<VEC> whole = {parts[buf][kWarps - 1][at.lane].a, back[buf][kWarps - 1][at.lane]};
#pragma unroll
      for (int j = kWarps - 2; j >= 0; --j) whole = joined<CUT>(whole, Run<VEC>{parts[buf][j][at.lane].a, back[buf][j][at.lane]});
      for (int r = at.warp; r < split; r += kWarps) store_cluster(tc::map_to_cta(tc::smem_u32(&tiles[buf][at.rank][at.lane]), (uint32_t)r), whole);
      __syncwarp();
      tc::cluster_sync_all();
      V behind = d;
#pragma unroll 4
      for (int r = split - 1; r >= 0; --r) {
        if (r == at.rank) behind = d;
        d = after<CUT>(tiles[buf][r][at.lane], d);
      }
      carry = d;
      d = behind;
    }
    V end = d;
    if (warps == kWarps) {
      V h = start;
#pragma unroll
      for (int j = 0; j < kWarps; ++j) {
        if (j == at.part) start = h;
        if (j + 1 < kWarps) h = after<CUT>(parts[buf][j][at.lane], h);
      }
#pragma unroll
      for (int j = kWarps - 1; j >= 0; --j) {
        if (j == at.part) end = d;
        d = after<CUT>(Run<VEC>{parts[buf][j][at.lane].a, back[buf][j][at.lane]}, d);
      }
    } else if (warps > 1) {
      for (int j = 0; j < at.part; ++j) start = after<CUT>(parts[buf][at.first + j][at.lane], start);
      for (int j = warps - 1; j >= 0; --j) {
        if (j == at.part) end = d;
        d = after<CUT>(Run<VEC>{parts[buf][at.first + j][at.lane].a, back[buf][at.first + j][at.lane]}, d);
      }
    } else {
      d = after<CUT>(Run<VEC>{sum.a, up}, d);
    }
    if (split == 1) carry = d;
    // the states in front of each step, then dh from the last step to the first
    V before[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      before[i] = start;
      if (CUT && (cuts >> i & 1)) before[i] = all<VEC>(0.f);
      start = fma(f[i], before[i], mul(GATE ? u[GATE ? i : 0] : n[i], x_of(i)));
    }
    const int rows = at.live ? a.steps - t0 : 0;
    const long long out = ((long long)at.b * a.steps + t0 + STEPS - 1) * a.channels + at.c;
    T *to_x = static_cast<T*>(g.dx) + out, *to_f = static_cast<T*>(g.dforget) + out, *to_i = static_cast<T*>(g.dinput) + (GATE ? out : 0);
#pragma unroll
    for (int i = STEPS - 1; i >= 0; --i) {
      const V x = x_of(i), dh = add(end, dy_of(i));
      const V dx = mul(dh, GATE ? u[GATE ? i : 0] : n[i]);
      const V df = mul(mul(dh, GATE ? before[i] : fma(x, all<VEC>(-1.f), before[i])), mul(f[i], n[i]));
      end = mul(f[i], dh);
      if (CUT && (cuts >> i & 1)) end = all<VEC>(0.f);
      if (i < rows) {
        L::store(to_x, dx);
        L::store(to_f, df);
        if constexpr (GATE) L::store(to_i, mul(mul(dh, x), mul(u[i], m[i])));
      }
      to_x -= a.channels;
      to_f -= a.channels;
      if constexpr (GATE) to_i -= a.channels;
    }
    __syncwarp();                              // the slot has been read
  }
  wait_copies<0>();
  if (at.rank == 0 && at.part == 0 && at.live) store_f(g.dstate + state_at, carry);
}

// How a call is laid out: a warp alone on its channels where that makes kBusy warps for every SM; else more warps side by side in time; else
// clusters. The backward pass's part of this decides what the forward pass keeps, so it goes by sizes alone.
constexpr long long kBusy = 16;
struct Shape { int warps, split, threads; unsigned blocks; };
int warps_of(const ScanArgs& a, int steps) {
  const long long columns = (long long)a.batch * ((a.channels + 63) / 64), runs = (a.steps + steps - 1) / steps;
  int warps = 1;
  while (warps < kWarps && warps < runs && columns * warps < kBusy * sm_count()) warps *= 2;
  return warps;
}
Shape shape_of(const ScanArgs& a, int vec, int steps) {
  const long long columns = (long long)a.batch * ((a.channels + 32 * vec - 1) / (32 * vec));
  Shape s;
  s.warps = warps_of(a, steps);
  const int beside = kWarps / s.warps;
  s.threads = 32 * kWarps;
  s.split = 1;
  const long long tiles = (a.steps + s.warps * steps - 1) / (s.warps * steps);
  if (s.warps == kWarps)
    while (s.split < kMostSplit && tiles >= 2 * s.split && columns * s.split * kWarps < kBusy * sm_count()) s.split *= 2;
  s.blocks = (unsigned)((columns + beside - 1) / beside * s.split);
  return s;
}

template <typename... K, typename... A>
cudaError_t launch(void (*kernel)(K...), const Shape& s, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.blocks);
  cfg.blockDim = dim3(s.threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)s.split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = s.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args..., s.warps, s.split);
}
// More shared memory than a kernel has by itself, and clusters of more than 8 blocks, have to be asked for, once per kernel.
template <class Kernel>
cudaError_t allow(Kernel kernel, size_t smem) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  return e != cudaSuccess ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}

int tile_of(const ScanArgs& a) { return warps_of(a, kBack) * kBack; }

template <typename T, int VEC, bool GATE, bool CUT, int STEPS>
cudaError_t run_forward(const ScanArgs& a, void* y, float* last, float* kept, int wide, cudaStream_t st) {
  auto kernel = scan_fwd_kernel<T, VEC, GATE, CUT, STEPS>;
  constexpr size_t smem = kWarps * Ring<T, VEC, STEPS, GATE ? 3 : 2>::BYTES;
  static const cudaError_t allowed = allow(kernel, smem);
  if (allowed != cudaSuccess) return allowed;
  const Shape s = shape_of(a, VEC, STEPS);
  return launch(kernel, s, smem, st, a, static_cast<T*>(y), last, kept, tile_of(a), wide);
}
template <typename T, int VEC, bool GATE, bool CUT>
cudaError_t run_backward(const ScanArgs& a, const ScanGrads& g, int wide, cudaStream_t st) {
  auto kernel = scan_bwd_kernel<T, VEC, GATE, CUT>;
  constexpr size_t smem = kWarps * Ring<T, VEC, kBack, GATE ? 4 : 3>::BYTES;
  static const cudaError_t allowed = allow(kernel, smem);
  if (allowed != cudaSuccess) return allowed;
  return launch(kernel, shape_of(a, VEC, kBack), smem, st, a, g, wide);
}
template <typename T, int VEC, int STEPS>
cudaError_t forward(const ScanArgs& a, void* y, float* last, float* kept, int wide, cudaStream_t st) {
  if (a.reset != nullptr)
    return a.input.p != nullptr ? run_forward<T, VEC, true, true, STEPS>(a, y, last, kept, wide, st) : run_forward<T, VEC, false, true, STEPS>(a, y, last, kept, wide, st);
  return a.input.p != nullptr ? run_forward<T, VEC, true, false, STEPS>(a, y, last, kept, wide, st) : run_forward<T, VEC, false, false, STEPS>(a, y, last, kept, wide, st);
}
template <typename T, int VEC>
cudaError_t backward(const ScanArgs& a, const ScanGrads& g, int wide, cudaStream_t st) {
  if (a.reset != nullptr) return a.input.p != nullptr ? run_backward<T, VEC, true, true>(a, g, wide, st) : run_backward<T, VEC, false, true>(a, g, wide, st);
  return a.input.p != nullptr ? run_backward<T, VEC, true, false>(a, g, wide, st) : run_backward<T, VEC, false, false>(a, g, wide, st);
}

// Whether all views' rows start on multiples of `bytes` and hold whole pieces of as many.
bool rows_fit(const ScanArgs& a, int bytes, std::initializer_list<ScanView> views) {
  const int size = a.bf16 ? 2 : 4;
  if (a.channels * size % bytes != 0) return false;
  for (const ScanView& v : views)
    if (v.p != nullptr && (reinterpret_cast<uintptr_t>(v.p) % bytes != 0 || v.batch * size % bytes != 0 || v.step * size % bytes != 0)) return false;
  return true;
}
bool floats_in_pairs(std::initializer_list<const float*> vectors) {
  for (const float* v : vectors)
    if (reinterpret_cast<uintptr_t>(v) % 8 != 0) return false;
  return true;
}

}  // namespace

int gated_scan_tile(const ScanArgs& a) { return tile_of(a); }

cudaError_t gated_scan_fwd(const ScanArgs& a, void* y, float* last, float* kept, cudaStream_t st) {
  if (a.batch <= 0 || a.channels <= 0) return cudaSuccess;
  const bool pairs = rows_fit(a, a.bf16 ? 4 : 8, {a.x, a.forget, a.input}) && floats_in_pairs({a.state, last, kept});
  const int wide = rows_fit(a, 16, {a.x, a.forget, a.input});
  if (!a.bf16) return pairs ? forward<float, 2, 8>(a, y, last, kept, wide, st) : forward<float, 1, 8>(a, y, last, kept, wide, st);
  if (!pairs) return forward<bf16, 1, 8>(a, y, last, kept, wide, st);
  return a.input.p == nullptr && a.steps >= 16 * kWarps ? forward<bf16, 2, 16>(a, y, last, kept, wide, st) : forward<bf16, 2, 8>(a, y, last, kept, wide, st);
}
cudaError_t gated_scan_bwd(const ScanArgs& a, const ScanGrads& g, cudaStream_t st) {
  if (a.batch <= 0 || a.channels <= 0) return cudaSuccess;
  const bool pairs = rows_fit(a, a.bf16 ? 4 : 8, {a.x, a.forget, a.input, g.dy}) && floats_in_pairs({g.kept, g.dlast, g.dstate});
  const int wide = rows_fit(a, 16, {a.x, a.forget, a.input, g.dy});
  if (!a.bf16) return pairs ? backward<float, 2>(a, g, wide, st) : backward<float, 1>(a, g, wide, st);
  return pairs ? backward<bf16, 2>(a, g, wide, st) : backward<bf16, 1>(a, g, wide, st);
}

}  // namespace adb200
