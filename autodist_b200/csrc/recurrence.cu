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
//   chunks          of the sequence go to blocks of their own where there are fewer still. What the chunks do is computed first, by a kernel
//                   whose warps hear from nobody (the inputs are read twice, but by as many blocks as the GPU holds); a chunk's block
//                   folds those in front of its own. The order of joining is fixed.
//
// Measured (B200, replayed back to back, bf16; share of the copy rate by the bytes that have to move): 32 x 2048 x 1024 forward 72 us (0.85),
// backward 136 (0.75); 1 x 65536 x 1024 127 (0.48; its inputs are read twice) and 182 (0.56); 128 x 20 x 2048 with an input gate 12.8
// (0.50) and 18.7 (0.60); in fp32 1 x 32768 x 1024 108 and 152. What bounds them is issuing instructions, 19 a value forward and 39
// backward, of which the memory would allow 33 and 55 with every issue slot taken: so values go in pairs, gates stay in registers
// (8 or 16 steps of a warp: what 128 registers hold at 16 warps an SM), and inputs are read again from shared memory instead of
// being kept (32 x 2048 x 1024 backward 156 -> 136).
//
// The states are not stored: the forward pass keeps them in fp32 in front of every tile of the backward pass, which walks the other way with
// the same joining of dh and computes those in between again. States, gates and sums are fp32.
#include "recurrence.h"

#include <cuda_bf16.h>

#include <initializer_list>
#include <type_traits>

#include "pdl.cuh"
#include "sm_count.h"
#include "tcgen05_common.cuh"

namespace adb200 {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int kWarps = 8;                    // of a block at most
constexpr int kBack = 8;                     // steps of a warp in the backward pass
constexpr int kLeastTiles = 2;               // of a chunk

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
// 1 / (1 + e). NEWTON, for the forget gates: a step of Newton's, without which products of a thousand gates close to one show a bias of the
// approximation's last bit (1 x 65536 x 1024: the state's gradient 1.0e-6 off, 0.6e-6 with it). In single values: in pairs it cost
// the backward pass 18 % of its time in registers moved about (32 x 2048 x 1024 132 -> 156 us, in single values 136).
template <bool NEWTON, int VEC> __device__ __forceinline__ F<VEC> reciprocal(F<VEC> e) {
  return each(add(e, all<VEC>(1.f)), [](float d) {
    const float r = rcp_fast(d);
    return NEWTON ? fmaf(r, fmaf(-d, r, 1.f), r) : r;
  });
}
template <typename T, int VEC, bool NEWTON> struct Gate;
template <int VEC, bool NEWTON> struct Gate<bf16, VEC, NEWTON> {
  F<VEC> bias;
  __device__ __forceinline__ explicit Gate(float b) : bias(all<VEC>(-kLog2e * b)) {}
  __device__ __forceinline__ void operator()(F<VEC> g, F<VEC>& f, F<VEC>& n) const {
    const F<VEC> e = each(fma(g, all<VEC>(-kLog2e), bias), [](float x) { return exp2_fast(min_nan(x, 126.f)); });
    f = reciprocal<NEWTON>(e);
    n = mul(e, f);
  }
};
template <int VEC, bool NEWTON> struct Gate<float, VEC, NEWTON> {
  F<VEC> bias;
  __device__ __forceinline__ explicit Gate(float b) : bias(all<VEC>(b)) {}
  __device__ __forceinline__ void operator()(F<VEC> g, F<VEC>& f, F<VEC>& n) const {
    const F<VEC> z = each(add(g, bias), [](float x) { return min_nan(max_nan(x, -87.f), 110.f); });
    const F<VEC> x = mul(z, all<VEC>(-kLog2e));
    const F<VEC> cut = fma(z, all<VEC>(-1.925963033500e-08f), fma(z, all<VEC>(-kLog2e), mul(x, all<VEC>(-1.f))));     // log2(e) is kLog2e + 1.926e-8
    const F<VEC> p = each(x, exp2_fast);
    const F<VEC> e = fma(p, mul(cut, all<VEC>(0.69314718f)), p);
    f = reciprocal<NEWTON>(e);
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

// Where a thread works. `warps`: warps of a tile; a block holds kWarps / warps tiles of neighbouring channel groups, or one.
template <int VEC>
struct Place {
  int lane, warp, part, first;               // part: the warp's place in its tile, whose first warp is `first`
  int b, c0, c, chunk;                       // c0: the warp's first channel
  bool live;
  __device__ __forceinline__ Place(const ScanArgs& a, int warps, int chunks) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    part = warp % warps;
    first = warp - part;
    chunk = blockIdx.x % chunks;
    const int across = (a.channels + 32 * VEC - 1) / (32 * VEC);
    const int column = blockIdx.x / chunks * (blockDim.x / 32 / warps) + warp / warps;
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
  static constexpr int FIT = 94 * 1024 / (kWarps * SLOT);       // two blocks and what they exchange through on an SM
  static constexpr int SLOTS = FIT < 2 ? 2 : FIT > 4 ? 4 : FIT;
  static constexpr int BYTES = SLOTS * SLOT;             // of a warp
};

// One tensor's rows of a warp, from which it requests a tile after the other. `wide`: whole 16-byte pieces, else a lane's channels by itself.
template <typename T, int VEC, int STEPS>
struct Source {
  typedef typename Lane<T, VEC>::Raw Raw;
  static constexpr int ROW = 32 * VEC * (int)sizeof(T), PIECES = ROW / 16, PER = 32 / PIECES;
  static_assert(STEPS % PER == 0, "whole rounds of pieces");
  const T* src;                              // what this lane copies first
  long long step, advance;                   // from a step to the next, and from a request to the next
  __device__ __forceinline__ Source(const ScanView& v, int b, int t0, int c0, int lane, bool wide, int steps_between) {
    src = static_cast<const T*>(v.p) + b * v.batch + t0 * v.step + c0 + (wide ? lane / PIECES * v.step + lane % PIECES * (16 / (int)sizeof(T)) : lane * VEC);
    step = v.step;
    advance = steps_between * v.step;
  }
  // Rows and channels that are not there hold `none`. `full`: all of them are.
  __device__ __forceinline__ void request(uint8_t* dst, int rows, int channels, int lane, bool wide, bool full, Raw none) {
    const T* from = src;
    src += advance;
    if (wide && full) {
      const uint32_t to = tc::smem_u32(dst) + (uint32_t)lane * 16u;
#pragma unroll
      for (int i = 0; i < STEPS / PER; ++i, from += PER * step) copy_async<16>(to + i * 512u, from);
    } else if (wide) {
      uint8_t* to = dst + lane * 16;
      const int left = lane % PIECES * (16 / (int)sizeof(T)) < channels ? rows - lane / PIECES : 0;
#pragma unroll 1
      for (int i = 0; i < STEPS / PER; ++i, from += PER * step, to += 512) {
        if (i * PER < left) {
          copy_async<16>(tc::smem_u32(to), from);
        } else {
          for (int j = 0; j < 16 / (int)sizeof(Raw); ++j) reinterpret_cast<Raw*>(to)[j] = none;
        }
      }
    } else {
      Raw* to = reinterpret_cast<Raw*>(dst) + lane;
      const int left = lane * VEC < channels ? rows : 0;
#pragma unroll
      for (int i = 0; i < STEPS; ++i, from += step, to += 32) {
        if (i < left) {
          if constexpr (sizeof(Raw) >= 4) copy_async<sizeof(Raw)>(tc::smem_u32(to), from);
          else *to = *reinterpret_cast<const Raw*>(from);
        } else {
          *to = none;
        }
      }
    }
  }
};
// A lane's place in rows that are `row` bytes apart.
template <typename T> __device__ __forceinline__ T* row_at(T* p, uint32_t row, uint32_t i) {
  return reinterpret_cast<T*>(reinterpret_cast<char*>(p) + (uint64_t)row * i);
}
// Bit i: the state in front of step t0 + i is forgotten.
template <int STEPS>
__device__ __forceinline__ uint32_t load_cuts(const ScanArgs& a, int b, int t0, int lane) {
  const bool cut = lane < STEPS && b < a.batch && t0 >= 0 && t0 + lane < a.steps && a.reset[b * a.reset_batch + (long long)(t0 + lane) * a.reset_step] != 0;
  return __ballot_sync(0xffffffffu, cut);
}

// A few steps, a single token among them: a thread walks through its channels' by itself.
constexpr int kFew = 4;
template <typename T, int VEC, bool GATE>
__global__ void __launch_bounds__(256) scan_few_kernel(const ScanArgs a, T* __restrict__ y, float* __restrict__ last, float* __restrict__ kept) {
  typedef Lane<T, VEC> L;
  typedef F<VEC> V;
  pdl_sync();
  const int across = a.channels / VEC;
  const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (at >= (long long)across * a.batch) return;
  const int b = (int)(at / across), c = (int)(at % across) * VEC;
  const long long state_at = (long long)b * a.channels + c;
  V h = a.state != nullptr ? load_f(a.state + state_at, static_cast<V*>(nullptr)) : all<VEC>(0.f);
  if (kept != nullptr && a.steps > 0) store_f(kept + state_at, h);            // all steps lie in one tile
  const Gate<T, VEC, true> forget(a.forget_bias);
  const Gate<T, VEC, false> input(0.f);
  auto read = [&](const ScanView& v, int t) { return L::unpack(*reinterpret_cast<const typename L::Raw*>(static_cast<const T*>(v.p) + b * v.batch + t * v.step + c)); };
  for (int t = 0; t < a.steps; ++t) {
    V f, n;
    forget(read(a.forget, t), f, n);
    if constexpr (GATE) {
      V m;
      input(read(a.input, t), n, m);
    }
    const V w = mul(n, read(a.x, t));
    const bool cut = a.reset != nullptr && a.reset[b * a.reset_batch + t * a.reset_step] != 0;
    h = cut ? w : fma(f, h, w);
    L::store(y + ((long long)b * a.steps + t) * a.channels + c, h);
  }
  store_f(last + state_at, h);
}

// Chunks of `tiles` tiles each that a sequence is cut into. runs: what the `pieces` of each do to a state (forward) or to dh (backward),
// [count * pieces][2][batch][channels].
struct Chunks {
  int count, tiles, pieces;
  float* runs;
  template <int VEC> __device__ __forceinline__ Run<VEC> run(const ScanArgs& a, int z, long long state_at) const {
    const long long plane = (long long)a.batch * a.channels;
    const float* p = runs + 2LL * z * plane + state_at;
    return {load_f(p, static_cast<F<VEC>*>(nullptr)), load_f(p + plane, static_cast<F<VEC>*>(nullptr))};
  }
};

// What each piece of each chunk but the last (backward: but the first) does: its steps in equal runs, a warp each.
template <typename T, int VEC, bool GATE, bool CUT, bool BACK>
__global__ void __launch_bounds__(32 * kWarps, 3)
scan_chunks_kernel(const ScanArgs a, const ScanView dy, const int wide, const int tile_steps, const Chunks ch) {
  typedef Lane<T, VEC> L;
  constexpr int STEPS = kBack;
  constexpr bool INPUT = GATE && !BACK;
  typedef Ring<T, VEC, STEPS, INPUT ? 3 : 2> R;
  extern __shared__ __align__(16) uint8_t ring_all[];
  __shared__ Run<VEC> parts[kWarps][32];
  pdl_sync();
  const Place<VEC> at(a, kWarps, (ch.count - 1) * ch.pieces);
  const int chunk = at.chunk / ch.pieces + (BACK ? 1 : 0), piece = at.chunk % ch.pieces, z = chunk * ch.pieces + piece;
  const int tile0 = ch.tiles * piece / ch.pieces, run_steps = (ch.tiles * (piece + 1) / ch.pieces - tile0) * tile_steps / kWarps;
  const int t_first = (chunk * ch.tiles + tile0) * tile_steps + at.warp * run_steps, rounds = run_steps / STEPS;
  const int channels = a.channels - at.c0;
  uint8_t* ring = ring_all + at.warp * R::BYTES;
  Source<T, VEC, STEPS> from_forget(a.forget, at.b, t_first, at.c0, at.lane, wide, STEPS), from_value(BACK ? dy : a.x, at.b, t_first, at.c0, at.lane, wide, STEPS),
      from_input(a.input, at.b, t_first, at.c0, at.lane, wide, STEPS);
  int rows = a.steps - t_first;
  auto request = [&](int k) {
    if (k < rounds) {
      uint8_t* slot = ring + k % R::SLOTS * R::SLOT;
      const bool full = rows >= STEPS && channels >= 32 * VEC, value = !BACK || dy.p != nullptr;
      from_forget.request(slot, rows, channels, at.lane, wide, full, L::kOpen);
      from_value.request(slot + STEPS * R::ROW, value ? rows : 0, channels, at.lane, wide, full && value, 0);
      if constexpr (INPUT) from_input.request(slot + 2 * STEPS * R::ROW, rows, channels, at.lane, wide, full, 0);
      rows -= STEPS;
    }
    commit_copies();
  };
#pragma unroll
  for (int k = 0; k < R::SLOTS - 1; ++k) request(k);
  const Gate<T, VEC, true> forget(a.forget_bias);
  const Gate<T, VEC, false> input(0.f);
  uint32_t cuts = 0, next_cuts = 0;
  if (CUT) next_cuts = load_cuts<STEPS>(a, at.b, t_first, at.lane);
  Run<VEC> sum = {all<VEC>(1.f), all<VEC>(0.f)};
  for (int k = 0; k < rounds; ++k) {
    request(k + R::SLOTS - 1);
    wait_copies<R::SLOTS - 1>();
    __syncwarp();
    if (CUT) {
      cuts = next_cuts;
      if (k + 1 < rounds) next_cuts = load_cuts<STEPS>(a, at.b, t_first + (k + 1) * STEPS, at.lane);
    }
    const typename L::Raw* raw = reinterpret_cast<const typename L::Raw*>(ring + k % R::SLOTS * R::SLOT) + at.lane;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      F<VEC> f, n;
      forget(L::unpack(raw[i * 32]), f, n);
      if constexpr (INPUT) {
        F<VEC> m;
        input(L::unpack(raw[(2 * STEPS + i) * 32]), n, m);
      }
      const F<VEC> value = L::unpack(raw[(STEPS + i) * 32]);
      const bool cut = CUT && (cuts >> i & 1);
      if (BACK) {                              // f_0 (dy_0 + f_1 (dy_1 + ...)), summed from the front
        sum.a = mul(sum.a, f);
        if (cut) sum.a = all<VEC>(-0.f);
        const F<VEC> more = fma(sum.a, value, sum.b);
        sum.b = CUT ? where_cut(sum.a, sum.b, more) : more;
      } else {
        const F<VEC> w = mul(n, value);
        sum = {mul(sum.a, f), fma(f, sum.b, w)};
        if (cut) sum = {all<VEC>(-0.f), w};
      }
    }
    __syncwarp();                              // the slot has been read
  }
  wait_copies<0>();
  parts[at.warp][at.lane] = sum;
  __syncthreads();
  if (at.warp == 0 && at.live) {
    Run<VEC> whole = parts[BACK ? kWarps - 1 : 0][at.lane];
#pragma unroll
    for (int j = 1; j < kWarps; ++j) whole = joined<CUT>(whole, parts[BACK ? kWarps - 1 - j : j][at.lane]);
    const long long plane = (long long)a.batch * a.channels;
    float* p = ch.runs + 2LL * z * plane + (long long)at.b * a.channels + at.c;
    store_f(p, whole.a);
    store_f(p + plane, whole.b);
  }
}

template <typename T, int VEC, bool GATE, bool CUT, int STEPS>
__global__ void __launch_bounds__(32 * kWarps, 2)
scan_fwd_kernel(const ScanArgs a, T* __restrict__ y, float* __restrict__ last, float* __restrict__ kept, const int keep_log2, const int wide,
                const int warps, const Chunks ch) {
  typedef Lane<T, VEC> L;
  typedef F<VEC> V;
  typedef Ring<T, VEC, STEPS, GATE ? 3 : 2> R;
  extern __shared__ __align__(16) uint8_t ring_all[];
  __shared__ Run<VEC> parts[2][kWarps][32];
  __shared__ V carries[2][kWarps][32];         // the state behind a tile
  pdl_sync();
  const Place<VEC> at(a, warps, ch.count);
  const int tile_steps = warps * STEPS;
  const int count = (a.steps + tile_steps - 1) / tile_steps, tile0 = at.chunk * ch.tiles, rounds = min(ch.tiles, count - tile0);
  uint8_t* ring = ring_all + at.warp * R::BYTES;
  const bool there = at.b < a.batch;
  const int t_first = tile0 * tile_steps + at.part * STEPS;
  const int channels = there ? a.channels - at.c0 : 0;         // of this warp, from its first on
  Source<T, VEC, STEPS> from_forget(a.forget, at.b, t_first, at.c0, at.lane, wide, tile_steps), from_x(a.x, at.b, t_first, at.c0, at.lane, wide, tile_steps),
      from_input(a.input, at.b, t_first, at.c0, at.lane, wide, tile_steps);
  int request_rows = a.steps - t_first;
  auto request = [&](int k) {
    if (k < rounds) {
      uint8_t* slot = ring + k % R::SLOTS * R::SLOT;
      const bool full = request_rows >= STEPS && channels >= 32 * VEC;
      from_forget.request(slot, request_rows, channels, at.lane, wide, full, L::kOpen);
      from_x.request(slot + STEPS * R::ROW, request_rows, channels, at.lane, wide, full, 0);
      if constexpr (GATE) from_input.request(slot + 2 * STEPS * R::ROW, request_rows, channels, at.lane, wide, full, 0);
      request_rows -= tile_steps;
    }
    commit_copies();
  };
#pragma unroll
  for (int k = 0; k < R::SLOTS - 1; ++k) request(k);
  const long long state_at = (long long)at.b * a.channels + at.c;
  V carry = at.live && a.state != nullptr ? load_f(a.state + state_at, static_cast<V*>(nullptr)) : all<VEC>(0.f);
  if (at.live)
#pragma unroll 4
    for (int z = 0; z < at.chunk * ch.pieces; ++z) carry = after<CUT>(ch.run<VEC>(a, z, state_at), carry);
  const Gate<T, VEC, true> forget(a.forget_bias);
  const Gate<T, VEC, false> input(0.f);
  uint32_t cuts = 0, next_cuts = 0;
  if (CUT) next_cuts = load_cuts<STEPS>(a, at.b, t_first, at.lane);

  for (int k = 0; k < rounds; ++k) {
    const int t0 = t_first + k * tile_steps, buf = k & 1;
    request(k + R::SLOTS - 1);
    wait_copies<R::SLOTS - 1>();
    __syncwarp();
    if (CUT) {
      cuts = next_cuts;
      if (k + 1 < rounds) next_cuts = load_cuts<STEPS>(a, at.b, t0 + tile_steps, at.lane);
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
    V start = carry;
    if (warps > 1) {
      parts[buf][at.warp][at.lane] = sum;
      __syncthreads();
      if (k > 0) start = carries[buf ^ 1][at.first][at.lane];
#pragma unroll 4
      for (int j = 0; j < at.part; ++j) start = after<CUT>(parts[buf][at.first + j][at.lane], start);
      carry = after<CUT>(sum, start);          // the last warp knows what the next tile starts from
      if (at.part == warps - 1) carries[buf][at.first][at.lane] = carry;
    } else {
      carry = after<CUT>(sum, start);
    }
    const int rows = at.live ? a.steps - t0 : 0;
    // states in front of the backward pass's tiles
    auto keep_state = [&](int t, V h) {
      store_f(kept + ((long long)at.b * ((a.steps + (1 << keep_log2) - 1) >> keep_log2) + (t >> keep_log2)) * a.channels + at.c, h);
    };
    const bool keeps = kept != nullptr && (t0 & ((1 << keep_log2) - 1)) == 0;
    if (keeps && rows > 0) keep_state(t0, start);
    T* out = y + ((long long)at.b * a.steps + t0) * a.channels + at.c;
    const uint32_t row = (uint32_t)a.channels * (uint32_t)sizeof(T);
    V h = start;
    if (rows >= STEPS && !(STEPS > kBack && keeps && (1 << keep_log2) == kBack)) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        h = CUT && (cuts >> i & 1) ? w[i] : fma(f[i], h, w[i]);
        L::store(row_at(out, row, i), h);
      }
    } else {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        if (STEPS > kBack && i == kBack && keeps && (1 << keep_log2) == kBack && i < rows) keep_state(t0 + i, h);
        h = CUT && (cuts >> i & 1) ? w[i] : fma(f[i], h, w[i]);
        if (i < rows) L::store(row_at(out, row, i), h);
      }
    }
  }
  wait_copies<0>();
  if (at.chunk == ch.count - 1 && at.part == warps - 1 && at.live) store_f(last + state_at, carry);
}

template <typename T, int VEC, bool GATE, bool CUT>
__global__ void __launch_bounds__(32 * kWarps, 2)
scan_bwd_kernel(const ScanArgs a, const ScanGrads g, const int wide, const int warps, const Chunks ch) {
  typedef Lane<T, VEC> L;
  typedef F<VEC> V;
  constexpr int STEPS = kBack;
  typedef Ring<T, VEC, STEPS, GATE ? 4 : 3> R;
  extern __shared__ __align__(16) uint8_t ring_all[];
  __shared__ Run<VEC> parts[2][kWarps][32];              // of a warp's steps
  __shared__ V carries[2][kWarps][32];                   // f dh in front of a tile
  __shared__ V back[2][kWarps][32];                      // their dh: from the end of the steps to their front it is a dh + back
  pdl_sync();
  const Place<VEC> at(a, warps, ch.count);
  const int tile_steps = warps * STEPS;
  const int count = (a.steps + tile_steps - 1) / tile_steps, tile0 = at.chunk * ch.tiles, rounds = min(ch.tiles, count - tile0);
  uint8_t* ring = ring_all + at.warp * R::BYTES;
  const bool there = at.b < a.batch;
  // rounds are counted from the last tiles to the first
  auto t0_of = [&](int k) { return (tile0 + rounds - 1 - k) * tile_steps + at.part * STEPS; };
  const int t_first = t0_of(0);
  const int channels = there ? a.channels - at.c0 : 0;         // of this warp, from its first on
  Source<T, VEC, STEPS> from_forget(a.forget, at.b, t_first, at.c0, at.lane, wide, -tile_steps), from_x(a.x, at.b, t_first, at.c0, at.lane, wide, -tile_steps),
      from_dy(g.dy, at.b, t_first, at.c0, at.lane, wide, -tile_steps), from_input(a.input, at.b, t_first, at.c0, at.lane, wide, -tile_steps);
  int request_rows = a.steps - t_first;
  auto request = [&](int k) {
    if (k < rounds) {
      uint8_t* slot = ring + k % R::SLOTS * R::SLOT;
      const bool full = request_rows >= STEPS && channels >= 32 * VEC, dy = g.dy.p != nullptr;
      from_forget.request(slot, request_rows, channels, at.lane, wide, full, L::kOpen);
      from_x.request(slot + STEPS * R::ROW, request_rows, channels, at.lane, wide, full, 0);
      from_dy.request(slot + 2 * STEPS * R::ROW, dy ? request_rows : 0, channels, at.lane, wide, full && dy, 0);
      if constexpr (GATE) from_input.request(slot + 3 * STEPS * R::ROW, request_rows, channels, at.lane, wide, full, 0);
      request_rows += tile_steps;
    }
    commit_copies();
  };
  auto front_of = [&](int k) {
    const int tile = tile0 + rounds - 1 - k;
    return at.live && k < rounds ? load_f(g.kept + ((long long)at.b * count + tile) * a.channels + at.c, static_cast<V*>(nullptr)) : all<VEC>(0.f);
  };
#pragma unroll
  for (int k = 0; k < R::SLOTS - 1; ++k) request(k);
  const long long state_at = (long long)at.b * a.channels + at.c;
  // f_{t+1} dh_{t+1} at the end of what is left
  V carry = at.live && g.dlast != nullptr ? load_f(g.dlast + state_at, static_cast<V*>(nullptr)) : all<VEC>(0.f);
  if (at.live)
#pragma unroll 4
    for (int z = ch.count * ch.pieces - 1; z >= (at.chunk + 1) * ch.pieces; --z) carry = after<CUT>(ch.run<VEC>(a, z, state_at), carry);
  V next_front = front_of(0);
  const Gate<T, VEC, true> forget(a.forget_bias);
  const Gate<T, VEC, false> input(0.f);
  uint32_t cuts = 0, next_cuts = 0;
  if (CUT) next_cuts = load_cuts<STEPS>(a, at.b, t0_of(0), at.lane);

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
    // read again where they are needed again: registers are what limits this kernel
    auto x_of = [&](int i) { return L::unpack(raw[(STEPS + i) * 32]); };
    auto dy_of = [&](int i) { return L::unpack(raw[(2 * STEPS + i) * 32]); };
    V f[STEPS], n[STEPS], u[GATE ? STEPS : 1], m[GATE ? STEPS : 1];              // sigmoids and their complements
    Run<VEC> sum = {all<VEC>(1.f), all<VEC>(0.f)};
    V up = all<VEC>(0.f);                      // f_0 (dy_0 + f_1 (dy_1 + ...)), summed from the front
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      forget(L::unpack(raw[i * 32]), f[i], n[i]);
      if constexpr (GATE) input(L::unpack(raw[(3 * STEPS + i) * 32]), u[i], m[i]);
      const V w = mul(GATE ? u[GATE ? i : 0] : n[i], x_of(i));
      if (i == 0) sum = {f[0], w};
      else sum = {mul(sum.a, f[i]), fma(f[i], sum.b, w)};
      if (CUT && (cuts >> i & 1)) sum = {all<VEC>(-0.f), w};
      const V more = fma(sum.a, dy_of(i), up);
      up = CUT ? where_cut(sum.a, up, more) : more;
    }
    V end = carry;
    if (warps > 1) {
      parts[buf][at.warp][at.lane] = sum;
      back[buf][at.warp][at.lane] = up;
      __syncthreads();
      if (k > 0) end = carries[buf ^ 1][at.first][at.lane];
#pragma unroll 4
      for (int j = 0; j < at.part; ++j) start = after<CUT>(parts[buf][at.first + j][at.lane], start);
#pragma unroll 4
      for (int j = warps - 1; j > at.part; --j) end = after<CUT>(Run<VEC>{parts[buf][at.first + j][at.lane].a, back[buf][at.first + j][at.lane]}, end);
      carry = after<CUT>(Run<VEC>{sum.a, up}, end);        // the first warp knows what the tile in front of this one ends on
      if (at.part == 0) carries[buf][at.first][at.lane] = carry;
    } else {
      carry = after<CUT>(Run<VEC>{sum.a, up}, end);
    }
    // the states in front of each step, then dh from the last step to the first
    V before[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      before[i] = start;
      if (CUT && (cuts >> i & 1)) before[i] = all<VEC>(0.f);
      start = fma(f[i], before[i], mul(GATE ? u[GATE ? i : 0] : n[i], x_of(i)));
    }
    const int rows = at.live ? a.steps - t0 : 0;
    const long long out = ((long long)at.b * a.steps + t0) * a.channels + at.c;
    T *to_x = static_cast<T*>(g.dx) + out, *to_f = static_cast<T*>(g.dforget) + out, *to_i = static_cast<T*>(g.dinput) + (GATE ? out : 0);
    const uint32_t row = (uint32_t)a.channels * (uint32_t)sizeof(T);
    auto walk = [&](auto whole) {
#pragma unroll
      for (int i = STEPS - 1; i >= 0; --i) {
        const V x = x_of(i), dh = add(end, dy_of(i));
        const V dx = mul(dh, GATE ? u[GATE ? i : 0] : n[i]);
        const V df = mul(mul(dh, GATE ? before[i] : fma(x, all<VEC>(-1.f), before[i])), mul(f[i], n[i]));
        end = mul(f[i], dh);
        if (CUT && (cuts >> i & 1)) end = all<VEC>(0.f);
        if (whole.value || i < rows) {
          L::store(row_at(to_x, row, i), dx);
          L::store(row_at(to_f, row, i), df);
          if constexpr (GATE) L::store(row_at(to_i, row, i), mul(mul(dh, x), mul(u[i], m[i])));
        }
      }
    };
    if (rows >= STEPS) walk(std::true_type());
    else walk(std::false_type());
    __syncwarp();                              // the slot has been read
  }
  wait_copies<0>();
  if (at.chunk == 0 && at.part == 0 && at.live) store_f(g.dstate + state_at, carry);
}

// How a call is laid out: a warp alone on its channels where that makes kBusy warps for every SM; else more warps side by side in time; else
// chunks. The backward pass's part of the warps decides what the forward pass keeps, so it goes by sizes alone.
constexpr long long kBusy = 16;
constexpr int kResident = 2;                 // blocks on an SM
constexpr int kPieceBlocks = 3;              // of the kernel that goes ahead
int warps_of(const ScanArgs& a, int steps) {
  const long long columns = (long long)a.batch * ((a.channels + 63) / 64), runs = (a.steps + steps - 1) / steps;
  int warps = 1;
  while (warps < kWarps && warps < runs && columns * warps < kBusy * sm_count()) warps *= 2;
  return warps;
}
long long columns_of(const ScanArgs& a, int vec) { return (long long)a.batch * ((a.channels + 32 * vec - 1) / (32 * vec)); }
// As many chunks as make one block for every place on the SMs, and as many pieces of them for the kernel that goes ahead.
Chunks chunks_of(const ScanArgs& a, int vec, int warps, int steps, float* runs) {
  const long long columns = columns_of(a, vec);
  const int tiles = (a.steps + warps * steps - 1) / (warps * steps);
  long long count = warps == kWarps && runs != nullptr ? kResident * sm_count() / columns : 1;
  if (count > tiles / kLeastTiles) count = tiles / kLeastTiles;
  if (count < 2) return {1, tiles, 1, nullptr};
  const int each = (int)((tiles + count - 1) / count);
  count = (tiles + each - 1) / each;
  long long pieces = kPieceBlocks * sm_count() / (columns * (count - 1));
  if (pieces > 32 / (count - 1)) pieces = 32 / (count - 1);              // a block folds them one after the other
  return {(int)count, each, (int)(pieces < 1 ? 1 : pieces > each ? each : pieces), runs};
}

// More shared memory than a kernel has by itself has to be asked for, once per kernel.
template <class Kernel>
cudaError_t allow(Kernel kernel, size_t smem) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }

int tile_log2(const ScanArgs& a) {
  int log2 = 0;
  while (1 << log2 < warps_of(a, kBack) * kBack) ++log2;
  return log2;
}

template <typename T, int VEC, bool GATE, bool CUT, bool BACK>
cudaError_t run_chunks(const ScanArgs& a, const ScanView& dy, int wide, int tile_steps, const Chunks& ch, cudaStream_t st) {
  if (ch.count == 1) return cudaSuccess;
  auto kernel = scan_chunks_kernel<T, VEC, GATE, CUT, BACK>;
  constexpr size_t smem = kWarps * Ring<T, VEC, kBack, GATE && !BACK ? 3 : 2>::BYTES;
  static const cudaError_t allowed = allow(kernel, smem);
  if (allowed != cudaSuccess) return allowed;
  return launch_pdl(kernel, dim3((unsigned)(columns_of(a, VEC) * (ch.count - 1) * ch.pieces)), dim3(32 * kWarps), smem, st, a, dy, wide, tile_steps, ch);
}
template <typename T, int VEC, bool GATE, bool CUT, int STEPS>
cudaError_t run_forward(const ScanArgs& a, void* y, float* last, float* kept, float* runs, int wide, int* launched, cudaStream_t st) {
  auto kernel = scan_fwd_kernel<T, VEC, GATE, CUT, STEPS>;
  constexpr size_t smem = kWarps * Ring<T, VEC, STEPS, GATE ? 3 : 2>::BYTES;
  static const cudaError_t allowed = allow(kernel, smem);
  if (allowed != cudaSuccess) return allowed;
  const int warps = warps_of(a, STEPS), beside = kWarps / warps;
  const Chunks ch = chunks_of(a, VEC, warps, STEPS, runs);
  const cudaError_t e = run_chunks<T, VEC, GATE, CUT, false>(a, a.x, wide, warps * STEPS, ch, st);
  if (e != cudaSuccess) return e;
  *launched = ch.count > 1 ? 2 : 1;
  const unsigned blocks = (unsigned)((columns_of(a, VEC) + beside - 1) / beside * ch.count);
  return launch_pdl(kernel, dim3(blocks), dim3(32 * kWarps), smem, st, a, static_cast<T*>(y), last, kept, tile_log2(a), wide, warps, ch);
}
template <typename T, int VEC, bool GATE, bool CUT>
cudaError_t run_backward(const ScanArgs& a, const ScanGrads& g, float* runs, int wide, int* launched, cudaStream_t st) {
  auto kernel = scan_bwd_kernel<T, VEC, GATE, CUT>;
  constexpr size_t smem = kWarps * Ring<T, VEC, kBack, GATE ? 4 : 3>::BYTES;
  static const cudaError_t allowed = allow(kernel, smem);
  if (allowed != cudaSuccess) return allowed;
  const int warps = warps_of(a, kBack), beside = kWarps / warps;
  const Chunks ch = chunks_of(a, VEC, warps, kBack, runs);
  const cudaError_t e = run_chunks<T, VEC, GATE, CUT, true>(a, g.dy, wide, warps * kBack, ch, st);
  if (e != cudaSuccess) return e;
  *launched = ch.count > 1 ? 2 : 1;
  const unsigned blocks = (unsigned)((columns_of(a, VEC) + beside - 1) / beside * ch.count);
  return launch_pdl(kernel, dim3(blocks), dim3(32 * kWarps), smem, st, a, g, wide, warps, ch);
}

template <typename T, int VEC, int STEPS>
cudaError_t forward(const ScanArgs& a, void* y, float* last, float* kept, float* runs, int wide, int* launched, cudaStream_t st) {
  // 128 x 2048 channels with an input gate, us: 1 step 2.6, walked through the ring 6.7; 4 steps 4.7 and 7.3
  if (a.steps <= kFew) {
    const long long threads = (long long)(a.channels / VEC) * a.batch;
    *launched = 1;
    return launch_pdl(a.input.p != nullptr ? scan_few_kernel<T, VEC, true> : scan_few_kernel<T, VEC, false>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a,
                      static_cast<T*>(y), last, kept);
  }
  if (a.reset != nullptr)
    return a.input.p != nullptr ? run_forward<T, VEC, true, true, STEPS>(a, y, last, kept, runs, wide, launched, st) : run_forward<T, VEC, false, true, STEPS>(a, y, last, kept, runs, wide, launched, st);
  return a.input.p != nullptr ? run_forward<T, VEC, true, false, STEPS>(a, y, last, kept, runs, wide, launched, st) : run_forward<T, VEC, false, false, STEPS>(a, y, last, kept, runs, wide, launched, st);
}
template <typename T, int VEC>
cudaError_t backward(const ScanArgs& a, const ScanGrads& g, float* runs, int wide, int* launched, cudaStream_t st) {
  if (a.reset != nullptr) return a.input.p != nullptr ? run_backward<T, VEC, true, true>(a, g, runs, wide, launched, st) : run_backward<T, VEC, false, true>(a, g, runs, wide, launched, st);
  return a.input.p != nullptr ? run_backward<T, VEC, true, false>(a, g, runs, wide, launched, st) : run_backward<T, VEC, false, false>(a, g, runs, wide, launched, st);
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

long long gated_scan_runs(const ScanArgs& a) {
  if (warps_of(a, kBack) < kWarps) return 0;
  // columns * (count - 1) * pieces is at most kPieceBlocks * SMs, or pieces is 1 and columns * count at most kResident * SMs
  const long long columns = columns_of(a, 2), most = (kPieceBlocks + kResident) * sm_count() / columns;
  return kResident * sm_count() / columns < 2 || a.steps < 2 * kLeastTiles * kWarps * kBack ? 0 : 2 * 2 * most * a.batch * a.channels;
}
int gated_scan_tile(const ScanArgs& a) { return 1 << tile_log2(a); }

cudaError_t gated_scan_fwd(const ScanArgs& a, void* y, float* last, float* kept, float* runs, int* launched, cudaStream_t st) {
  *launched = 0;
  if (a.batch <= 0 || a.channels <= 0) return cudaSuccess;
  const bool pairs = rows_fit(a, a.bf16 ? 4 : 8, {a.x, a.forget, a.input}) && floats_in_pairs({a.state, last, kept, runs});
  const int wide = rows_fit(a, 16, {a.x, a.forget, a.input});
  const bool longer = a.steps >= 16 * kWarps;
  if (!a.bf16) {
    if (pairs) return forward<float, 2, 8>(a, y, last, kept, runs, wide, launched, st);
    return longer ? forward<float, 1, 16>(a, y, last, kept, runs, wide, launched, st) : forward<float, 1, 8>(a, y, last, kept, runs, wide, launched, st);
  }
  if (pairs) return longer && a.input.p == nullptr ? forward<bf16, 2, 16>(a, y, last, kept, runs, wide, launched, st) : forward<bf16, 2, 8>(a, y, last, kept, runs, wide, launched, st);
  return longer ? forward<bf16, 1, 16>(a, y, last, kept, runs, wide, launched, st) : forward<bf16, 1, 8>(a, y, last, kept, runs, wide, launched, st);
}
cudaError_t gated_scan_bwd(const ScanArgs& a, const ScanGrads& g, float* runs, int* launched, cudaStream_t st) {
  *launched = 0;
  if (a.batch <= 0 || a.channels <= 0) return cudaSuccess;
  const bool pairs = rows_fit(a, a.bf16 ? 4 : 8, {a.x, a.forget, a.input, g.dy}) && floats_in_pairs({g.kept, g.dlast, g.dstate, runs});
  const int wide = rows_fit(a, 16, {a.x, a.forget, a.input, g.dy});
  if (!a.bf16) return pairs ? backward<float, 2>(a, g, runs, wide, launched, st) : backward<float, 1>(a, g, runs, wide, launched, st);
  return pairs ? backward<bf16, 2>(a, g, runs, wide, launched, st) : backward<bf16, 1>(a, g, runs, wide, launched, st);
}

}  // namespace adb200
