// Python bindings of a recurrent language model's operators: argument checks, outputs, launches on the current stream of the tensors' GPU.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
#include <memory>
#include <string>
#include <utility>
#include <vector>

#include "adamw_list.h"
#include "gemm_8bit.h"
#include "recurrence.h"
#include "rms_norm.h"

namespace {

using at::Tensor;
using c10::optional;

// A tensor's shape and type for a message. Put together here: the library's stream operator for shapes crashed in this extension.
std::string shown(const Tensor& t) {
  std::string r = "[";
  for (int64_t d = 0; d < t.dim(); ++d) r += (d ? ", " : "") + std::to_string(t.size(d));
  return r + "] " + c10::toString(t.scalar_type());
}

void launched(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e)); }

cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

bool same_gpu(const Tensor& a, const Tensor& b) { return b.is_cuda() && b.device() == a.device(); }
void check_gpu(const Tensor& a, const optional<Tensor>& b, const char* name) {
  TORCH_CHECK(!b.has_value() || same_gpu(a, *b), name, ": tensors on one GPU needed");
}

// Whether a stream's type is bf16; fp32 is the other one.
bool is_bf16(const Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, name, ": bf16 or fp32 needed, got ", shown(t));
  return t.scalar_type() == at::kBFloat16;
}

// [..., width] as [rows, width] with unit stride along the width: a view where the strides allow it.
Tensor as_rows(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}
// From one row to the next; a single row's stride means nothing.
int64_t row_stride(const Tensor& rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

// ---------------------------------------------------------------------------------------------- norm
int64_t check_width(const Tensor& x, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, ": a tensor on a GPU needed");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, name, ": rows of at least one element needed");
  TORCH_CHECK(x.size(-1) < (1LL << 30), name, ": rows too wide");
  return x.size(-1);
}
void check_like(const Tensor& x, const optional<Tensor>& other, const char* name, const char* what) {
  if (!other.has_value()) return;
  TORCH_CHECK(same_gpu(x, *other), name, ": ", what, " must be on the input's GPU");
  TORCH_CHECK(other->sizes() == x.sizes() && other->scalar_type() == x.scalar_type(), name, ": ", what, " must have the input's shape and type, got ",
              shown(*other), " for ", shown(x));
}
Tensor check_weight(const Tensor& x, const Tensor& weight, const char* name) {
  TORCH_CHECK(same_gpu(x, weight), name, ": the weight must be on the input's GPU");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(-1), name, ": a weight for each column needed, got ", shown(weight), " for ", shown(x));
  TORCH_CHECK(weight.scalar_type() == at::kFloat || weight.scalar_type() == x.scalar_type(), name, ": the weight must be fp32 or of the input's type, got ", shown(weight));
  return weight.contiguous();
}

// ---------------------------------------------------------------------------------------------- gradients
// Kernels that backward passes launched: those run in the autograd engine, not through the counted calls.
std::atomic<int64_t> g_backward_kernels{0};
int64_t backward_kernels() { return g_backward_kernels.load(); }

// Gradients that can be differentiated themselves: the same expression in PyTorch operations, by `name` in autodist_b200.ops.lm.
template <typename... Args>
torch::autograd::variable_list differentiable(const char* name, size_t inputs, Args&&... args) {
  pybind11::gil_scoped_acquire gil;
  const auto found = pybind11::module_::import("autodist_b200.ops.lm").attr(name)(std::forward<Args>(args)...).template cast<std::vector<optional<Tensor>>>();
  torch::autograd::variable_list grads;
  for (const auto& g : found) grads.push_back(g.has_value() ? *g : Tensor());
  grads.resize(inputs);
  return grads;
}
optional<Tensor> some(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; }

struct NormInputs {                        // what the addresses in `rows` belong to
  Tensor x, res, weight, sum;
  adb200::NormRows rows{};
};
NormInputs norm_inputs(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& residual, double eps, const char* name) {
  const int64_t width = check_width(x, name);
  NormInputs in;
  in.rows.bf16 = is_bf16(x, name);
  check_like(x, residual, name, "the residual");
  if (weight.has_value()) {
    in.weight = check_weight(x, *weight, name);
    in.rows.weight = in.weight.data_ptr();
    in.rows.weight_bf16 = in.weight.scalar_type() == at::kBFloat16;
  }
  in.x = as_rows(x);
  in.rows.x = in.x.data_ptr();
  in.rows.x_ld = row_stride(in.x);
  if (residual.has_value()) {
    in.res = as_rows(*residual);
    in.rows.res = in.res.data_ptr();
    in.rows.res_ld = row_stride(in.res);
    in.sum = at::empty(x.sizes(), x.options());
    in.rows.sum = in.sum.data_ptr();
  }
  in.rows.rows = in.x.size(0);
  in.rows.width = (int)width;
  in.rows.eps = (float)eps;
  return in;
}

// -> (y, x + residual)
std::tuple<Tensor, optional<Tensor>> rms_norm_fwd(const Tensor& x, const Tensor& weight, const optional<Tensor>& residual, double eps) {
  TORCH_CHECK(x.is_cuda(), "rms_norm: a tensor on a GPU needed");
  const c10::cuda::CUDAGuard guard(x.device());
  NormInputs in = norm_inputs(x, weight, residual, eps, "rms_norm");
  Tensor y = at::empty(x.sizes(), x.options());
  launched(adb200::rms_norm_fwd(in.rows, y.data_ptr(), stream_of(x)), "rms_norm");
  return {y, residual.has_value() ? optional<Tensor>(in.sum) : c10::nullopt};
}

// -> (gradient of the input and of the residual, gradient of the weight, kernels launched)
std::tuple<Tensor, Tensor, int> rms_norm_bwd(const Tensor& dy, const optional<Tensor>& ds, const Tensor& s, const Tensor& weight, double eps) {
  const char* name = "rms_norm";
  TORCH_CHECK(s.is_cuda(), "rms_norm: a tensor on a GPU needed");
  const c10::cuda::CUDAGuard guard(s.device());
  const int64_t width = check_width(s, name);
  check_like(s, dy, name, "the gradient");
  check_like(s, ds, name, "the sum's gradient");
  adb200::NormGrad g{};
  g.bf16 = is_bf16(s, name);
  const Tensor w = check_weight(s, weight, name), rows = as_rows(s), dyr = as_rows(dy);
  Tensor dsr;
  g.dy = dyr.data_ptr(); g.dy_ld = row_stride(dyr);
  if (ds.has_value()) {
    dsr = as_rows(*ds);
    g.ds = dsr.data_ptr(); g.ds_ld = row_stride(dsr);
  }
  g.s = rows.data_ptr(); g.s_ld = row_stride(rows);
  g.weight = w.data_ptr(); g.weight_bf16 = w.scalar_type() == at::kBFloat16;
  g.rows = rows.size(0); g.width = (int)width; g.eps = (float)eps;
  Tensor dx = at::empty(s.sizes(), s.options()), dw = at::empty(w.sizes(), w.options());
  g.dx = dx.data_ptr(); g.dw = dw.data_ptr();
  Tensor part = at::empty({adb200::rms_norm_bwd_floats(g)}, s.options().dtype(at::kFloat));
  g.part = part.data_ptr<float>();
  int kernels = 0;
  launched(adb200::rms_norm_bwd(g, &kernels, stream_of(s)), name);
  return {dx, dw, kernels};
}

class NormFunction : public torch::autograd::Function<NormFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight, const optional<Tensor>& residual, double eps) {
    auto [y, sum] = rms_norm_fwd(x, weight, residual, eps);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({sum.has_value() ? *sum : x, weight});
    ctx->saved_data["eps"] = eps;
    return sum.has_value() ? torch::autograd::variable_list{y, *sum} : torch::autograd::variable_list{y};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool residual = grads.size() > 1;
    const Tensor ds = residual ? grads[1] : Tensor();
    const double eps = ctx->saved_data["eps"].toDouble();
    // the sum is the only place where x and the residual meet: both get its gradient
    if (!grads[0].defined()) return {ds, Tensor(), ds, Tensor()};
    if (at::GradMode::is_enabled()) {
      auto again = differentiable("_norm_again", 2, saved[0], saved[1], eps, grads[0], some(ds));
      return {again[0], again[1], residual ? again[0] : Tensor(), Tensor()};
    }
    auto [dx, dw, launches] = rms_norm_bwd(grads[0], some(ds), saved[0], saved[1], eps);
    g_backward_kernels += launches;
    return {dx, dw, residual ? dx : Tensor(), Tensor()};
  }
};
// -> (y, x + residual), with a gradient where one is recorded
std::tuple<Tensor, optional<Tensor>> rms_norm(const Tensor& x, const Tensor& weight, const optional<Tensor>& residual, double eps) {
  const auto out = NormFunction::apply(x, weight, residual, eps);
  return {out[0], out.size() > 1 ? optional<Tensor>(out[1]) : c10::nullopt};
}

// Codes of [..., width] whose rows start on 16-byte boundaries.
Tensor empty_codes(const Tensor& x) {
  std::vector<int64_t> shape = x.sizes().vec();
  const int64_t width = shape.back();
  shape.back() = (width + 15) / 16 * 16;
  Tensor t = at::empty(shape, x.options().dtype(at::kFloat8_e4m3fn));
  return shape.back() == width ? t : t.narrow(-1, 0, width);
}
std::tuple<Tensor, Tensor, optional<Tensor>> rows_8bit(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& residual, double eps,
                                                       const char* name) {
  TORCH_CHECK(x.is_cuda(), name, ": a tensor on a GPU needed");
  const c10::cuda::CUDAGuard guard(x.device());
  NormInputs in = norm_inputs(x, weight, residual, eps, name);
  Tensor codes = empty_codes(x), scales = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  launched(adb200::rms_norm_8bit(in.rows, codes.data_ptr(), (in.rows.width + 15) / 16 * 16, scales.data_ptr<float>(), stream_of(x)), name);
  return {codes, scales, residual.has_value() ? optional<Tensor>(in.sum) : c10::nullopt};
}
// -> (codes, scales, x + residual)
std::tuple<Tensor, Tensor, optional<Tensor>> rms_norm_8bit(const Tensor& x, const Tensor& weight, const optional<Tensor>& residual, double eps) {
  return rows_8bit(x, weight, residual, eps, "rms_norm_8bit");
}
std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  auto r = rows_8bit(x, c10::nullopt, c10::nullopt, 0.0, "quantize_rows");
  return {std::get<0>(r), std::get<1>(r)};
}

// ---------------------------------------------------------------------------------------------- product
// Rows of codes as the kernels read them: on 16-byte boundaries.
Tensor aligned_codes(const Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn && t.dim() >= 1, "linear_8bit: ", what, " must be float8_e4m3fn, got ", shown(t));
  TORCH_CHECK(t.size(-1) > 0 && t.size(-1) < (1LL << 30), "linear_8bit: ", what, " must have between 1 and 2^30 columns, got ", shown(t));
  Tensor r = as_rows(t);
  if (reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0 && row_stride(r) % 16 == 0 && row_stride(r) >= r.size(1)) return r;
  if (r.size(0) <= 1 && reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0) return r;
  return empty_codes(r).copy_(r);
}
Tensor aligned_floats(const Tensor& t) {
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
int64_t code_stride(const Tensor& r) { return r.size(0) > 1 ? r.stride(0) : (r.size(1) + 15) / 16 * 16; }

// `bn`, `split`: see gemm_8bit.h
Tensor gemm_8bit(const Tensor& codes, const Tensor& scales, const Tensor& weight_codes, const Tensor& weight_scales, const optional<Tensor>& bias, Tensor error,
                 int64_t bn, int64_t split) {
  const char* name = "linear_8bit";
  TORCH_CHECK(codes.is_cuda(), "linear_8bit: tensors on a GPU needed");
  check_gpu(codes, scales, name); check_gpu(codes, weight_codes, name); check_gpu(codes, weight_scales, name); check_gpu(codes, bias, name);
  check_gpu(codes, error, name);
  const c10::cuda::CUDAGuard guard(codes.device());
  TORCH_CHECK(weight_codes.dim() == 2 && codes.size(-1) == weight_codes.size(1), "linear_8bit: rows of ", shown(codes), " and weights of ", shown(weight_codes),
              " do not match");
  const Tensor x = aligned_codes(codes, "the rows"), w = aligned_codes(weight_codes, "the weight");
  const int64_t M = x.size(0), N = w.size(0);
  TORCH_CHECK(M < (1LL << 31) && N < (1LL << 31), "linear_8bit: too many rows");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.sizes() == codes.sizes().slice(0, codes.dim() - 1) && weight_scales.dim() == 1 && weight_scales.scalar_type() == at::kFloat && weight_scales.numel() == N,
              "linear_8bit: an fp32 scale for each row needed");
  TORCH_CHECK(!bias.has_value() || (bias->scalar_type() == at::kFloat && bias->numel() == N), "linear_8bit: an fp32 bias for each output needed");
  TORCH_CHECK(error.scalar_type() == at::kInt && error.numel() >= 1, "linear_8bit: an int32 word needed");
  const Tensor sx = aligned_floats(scales), sw = aligned_floats(weight_scales), b = bias.has_value() ? aligned_floats(*bias) : Tensor();
  std::vector<int64_t> shape = codes.sizes().vec();
  shape.back() = N;
  Tensor y = at::empty(shape, codes.options().dtype(at::kBFloat16));
  adb200::Gemm8Args a{};
  a.codes = static_cast<const uint8_t*>(x.data_ptr()); a.codes_ld = code_stride(x);
  a.scales = sx.data_ptr<float>();
  a.weight_codes = static_cast<const uint8_t*>(w.data_ptr()); a.weight_ld = code_stride(w);
  a.weight_scales = sw.data_ptr<float>();
  a.bias = b.defined() ? b.data_ptr<float>() : nullptr;
  a.y = y.data_ptr();
  a.M = (int)M; a.N = (int)N; a.K = (int)x.size(1);
  a.error = error.data_ptr<int>();
  launched(adb200::gemm_8bit(a, (int)bn, (int)split, stream_of(codes)), name);
  return y;
}

// ---------------------------------------------------------------------------------------------- recurrence
struct ScanInputs {                        // what the addresses in `a` belong to
  Tensor x, forget, input, state, reset;
  adb200::ScanArgs a{};
};
adb200::ScanView scan_view(const Tensor& t, Tensor& held) {
  held = t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous();
  return {held.data_ptr(), held.stride(0), held.stride(1)};
}
ScanInputs scan_inputs(const Tensor& x, const Tensor& forget, const optional<Tensor>& input, const optional<Tensor>& state, const optional<Tensor>& reset,
                       double forget_bias) {
  const char* name = "gated_recurrence";
  TORCH_CHECK(x.dim() == 3, "gated_recurrence: [batch, steps, channels] needed, got ", shown(x));
  ScanInputs in;
  in.a.bf16 = is_bf16(x, name);
  check_like(x, forget, name, "the forget gate");
  check_like(x, input, name, "the input gate");
  const int64_t B = x.size(0), T = x.size(1), C = x.size(2);
  TORCH_CHECK(T < (1LL << 30) && B * ((C + 31) / 32) < (1LL << 31) / 64, "gated_recurrence: too large");
  in.a.x = scan_view(x, in.x);
  in.a.forget = scan_view(forget, in.forget);
  if (input.has_value()) in.a.input = scan_view(*input, in.input);
  if (state.has_value()) {
    TORCH_CHECK(same_gpu(x, *state) && state->scalar_type() == at::kFloat && state->dim() == 2 && state->size(0) == B && state->size(1) == C,
                "gated_recurrence: an fp32 state [batch, channels] on the input's GPU needed, got ", shown(*state));
    in.state = state->contiguous();
    in.a.state = in.state.data_ptr<float>();
  }
  if (reset.has_value()) {
    TORCH_CHECK(same_gpu(x, *reset) && reset->scalar_type() == at::kBool && reset->dim() == 2 && reset->size(0) == B && reset->size(1) == T,
                "gated_recurrence: a bool reset [batch, steps] on the input's GPU needed, got ", shown(*reset));
    in.reset = *reset;
    in.a.reset = static_cast<const uint8_t*>(reset->data_ptr());
    in.a.reset_batch = reset->stride(0);
    in.a.reset_step = reset->stride(1);
  }
  in.a.batch = (int)B; in.a.steps = (int)T; in.a.channels = (int)C;
  in.a.forget_bias = (float)forget_bias;
  return in;
}

int64_t kept_tiles(const adb200::ScanArgs& a) {
  const int64_t tile = adb200::gated_scan_tile(a);
  return (a.steps + tile - 1) / tile;
}

Tensor scan_scratch(const adb200::ScanArgs& a, const at::TensorOptions& f32) {
  const long long n = adb200::gated_scan_runs(a);
  return n > 0 ? at::empty({n}, f32) : Tensor();
}

// -> (outputs, last state, states kept for the backward pass, kernels launched)
std::tuple<Tensor, Tensor, optional<Tensor>, int> gated_scan_fwd(const Tensor& x, const Tensor& forget, const optional<Tensor>& input, const optional<Tensor>& state,
                                                            const optional<Tensor>& reset, double forget_bias, bool keep) {
  TORCH_CHECK(x.is_cuda(), "gated_recurrence: tensors on a GPU needed");
  const c10::cuda::CUDAGuard guard(x.device());
  ScanInputs in = scan_inputs(x, forget, input, state, reset, forget_bias);
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor y = at::empty(x.sizes(), x.options()), last = at::empty({x.size(0), x.size(2)}, f32), kept;
  if (keep) kept = at::empty({x.size(0), kept_tiles(in.a), x.size(2)}, f32);
  const Tensor runs = scan_scratch(in.a, f32);
  int kernels = 0;
  launched(adb200::gated_scan_fwd(in.a, y.data_ptr(), last.data_ptr<float>(), keep ? kept.data_ptr<float>() : nullptr, runs.defined() ? runs.data_ptr<float>() : nullptr,
                                  &kernels, stream_of(x)), "gated_recurrence");
  return {y, last, keep ? optional<Tensor>(kept) : c10::nullopt, kernels};
}

// -> gradients of (x, forget, input, state), kernels launched
std::tuple<Tensor, Tensor, optional<Tensor>, Tensor, int> gated_scan_bwd(const optional<Tensor>& dy, const optional<Tensor>& dlast, const Tensor& x, const Tensor& forget,
                                                                    const optional<Tensor>& input, const optional<Tensor>& state, const optional<Tensor>& reset,
                                                                    const Tensor& kept, double forget_bias) {
  TORCH_CHECK(x.is_cuda(), "gated_recurrence: tensors on a GPU needed");
  const c10::cuda::CUDAGuard guard(x.device());
  ScanInputs in = scan_inputs(x, forget, input, state, reset, forget_bias);
  check_like(x, dy, "gated_recurrence", "the gradient");
  const int64_t B = x.size(0), C = x.size(2);
  TORCH_CHECK(same_gpu(x, kept) && kept.scalar_type() == at::kFloat && kept.is_contiguous() &&
                  kept.numel() == B * C * kept_tiles(in.a), "gated_recurrence: the forward pass's states needed");
  adb200::ScanGrads g{};
  Tensor dy_held, dlast_held;
  if (dy.has_value()) g.dy = scan_view(*dy, dy_held);
  if (dlast.has_value()) {
    TORCH_CHECK(same_gpu(x, *dlast) && dlast->scalar_type() == at::kFloat && dlast->numel() == B * C, "gated_recurrence: an fp32 gradient of the last state needed");
    dlast_held = dlast->contiguous();
    g.dlast = dlast_held.data_ptr<float>();
  }
  Tensor dx = at::empty(x.sizes(), x.options()), dforget = at::empty(x.sizes(), x.options()), dstate = at::empty({B, C}, kept.options()), dinput;
  if (input.has_value()) dinput = at::empty(x.sizes(), x.options());
  g.kept = kept.data_ptr<float>();
  g.dx = dx.data_ptr(); g.dforget = dforget.data_ptr(); g.dinput = input.has_value() ? dinput.data_ptr() : nullptr; g.dstate = dstate.data_ptr<float>();
  const Tensor runs = scan_scratch(in.a, kept.options());
  int kernels = 0;
  launched(adb200::gated_scan_bwd(in.a, g, runs.defined() ? runs.data_ptr<float>() : nullptr, &kernels, stream_of(x)), "gated_recurrence");
  return {dx, dforget, input.has_value() ? optional<Tensor>(dinput) : c10::nullopt, dstate, kernels};
}

class ScanFunction : public torch::autograd::Function<ScanFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& forget, const optional<Tensor>& input,
                                                const optional<Tensor>& state, const optional<Tensor>& reset, double forget_bias, bool keep, int* kernels) {
    auto [y, last, kept, launches] = gated_scan_fwd(x, forget, input, state, reset, forget_bias, keep);
    *kernels = launches;
    if (keep) {
      ctx->set_materialize_grads(false);
      ctx->save_for_backward({x, forget, input.value_or(Tensor()), state.value_or(Tensor()), reset.value_or(Tensor()), *kept});
      ctx->saved_data["forget_bias"] = forget_bias;
    }
    return {y, last};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const double forget_bias = ctx->saved_data["forget_bias"].toDouble();
    torch::autograd::variable_list found;
    if (!grads[0].defined() && !grads[1].defined()) {
      found.resize(4);
    } else if (at::GradMode::is_enabled()) {
      found = differentiable("_scan_again", 4, saved[0], saved[1], some(saved[2]), some(saved[3]), some(saved[4]), forget_bias, some(grads[0]), some(grads[1]));
    } else {
      auto [dx, dforget, dinput, dstate, launches] = gated_scan_bwd(some(grads[0]), some(grads[1]), saved[0], saved[1], some(saved[2]), some(saved[3]), some(saved[4]),
                                                                    saved[5], forget_bias);
      g_backward_kernels += launches;
      found = {dx, dforget, dinput.value_or(Tensor()), saved[3].defined() ? dstate : Tensor()};
    }
    found.resize(8);
    return found;
  }
};
// -> (outputs, last state, kernels launched), with a gradient where one is recorded
std::tuple<Tensor, Tensor, int> gated_scan(const Tensor& x, const Tensor& forget, const optional<Tensor>& input, const optional<Tensor>& state,
                                           const optional<Tensor>& reset, double forget_bias) {
  const bool keep = at::GradMode::is_enabled() && (x.requires_grad() || forget.requires_grad() || (input.has_value() && input->requires_grad()) ||
                                                   (state.has_value() && state->requires_grad()));
  int kernels = 0;
  const auto out = ScanFunction::apply(x, forget, input, state, reset, forget_bias, keep, &kernels);
  return {out[0], out[1], kernels};
}

// ---------------------------------------------------------------------------------------------- optimizer
// The parameters of a group and where their moments lie. Addresses are read at every step: a parameter's storage may change.
struct AdamwList {
  std::vector<Tensor> params;
  std::vector<int64_t> places;             // first element of each parameter's moments
  Tensor m, r, m_scale, r_scale, step;
  uint64_t seed = 0;
};

std::shared_ptr<AdamwList> adamw_list(std::vector<Tensor> params, std::vector<int64_t> places, Tensor m, Tensor r, const optional<Tensor>& m_scale,
                                      const optional<Tensor>& r_scale, Tensor step, int64_t seed) {
  TORCH_CHECK(!params.empty() && params.size() == places.size(), "adamw: a place for each parameter needed");
  const bool bits8 = m_scale.has_value();
  const auto type = bits8 ? at::kFloat8_e4m3fn : at::kFloat;
  for (const Tensor* t : {&m, &r})
    TORCH_CHECK(same_gpu(params[0], *t) && t->scalar_type() == type && t->is_contiguous() && t->numel() % adb200::kAdamwBlock == 0, "adamw: bad moments");
  TORCH_CHECK(r.numel() == m.numel() && r_scale.has_value() == bits8, "adamw: bad moments");
  if (bits8)
    for (const Tensor* t : {&*m_scale, &*r_scale})
      TORCH_CHECK(same_gpu(params[0], *t) && t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == m.numel() / adb200::kAdamwBlock, "adamw: bad scales");
  TORCH_CHECK(same_gpu(params[0], step) && step.scalar_type() == at::kLong && step.is_contiguous() && step.numel() == 2, "adamw: a counter of two words needed");
  for (size_t i = 0; i < params.size(); ++i) {
    TORCH_CHECK(same_gpu(params[0], params[i]), "adamw: parameters on one GPU needed");
    is_bf16(params[i], "adamw");
    TORCH_CHECK(places[i] >= 0 && places[i] % adb200::kAdamwBlock == 0 && places[i] + params[i].numel() <= m.numel(), "adamw: a parameter's moments lie outside");
  }
  auto list = std::make_shared<AdamwList>();
  list->params = std::move(params);
  list->places = std::move(places);
  list->m = m; list->r = r;
  if (bits8) { list->m_scale = *m_scale; list->r_scale = *r_scale; }
  list->step = step;
  list->seed = (uint64_t)seed;
  return list;
}

// Each parameter's moments (and their scales) as views of the flat ones, the moments in the parameter's shape.
std::vector<std::vector<Tensor>> adamw_views(const std::shared_ptr<AdamwList>& l) {
  std::vector<std::vector<Tensor>> views;
  views.reserve(l->params.size());
  for (size_t i = 0; i < l->params.size(); ++i) {
    const Tensor& p = l->params[i];
    std::vector<int64_t> strides(p.dim());
    int64_t n = 1;
    for (int64_t d = p.dim() - 1; d >= 0; --d) { strides[d] = n; n *= p.size(d); }
    const int64_t block = l->places[i] / adb200::kAdamwBlock, blocks = (n + adb200::kAdamwBlock - 1) / adb200::kAdamwBlock;
    std::vector<Tensor> v{l->m.as_strided(p.sizes(), strides, l->places[i]), l->r.as_strided(p.sizes(), strides, l->places[i])};
    if (l->m_scale.defined()) {
      v.push_back(l->m_scale.narrow(0, block, blocks));
      v.push_back(l->r_scale.narrow(0, block, blocks));
    }
    views.push_back(std::move(v));
  }
  return views;
}

// One step over the parameters that have a gradient. Returns how many kernels it launched.
int64_t adamw_list_step(const std::shared_ptr<AdamwList>& l, double lr, const optional<Tensor>& lr_at, double b1, double b2, double eps, double wd) {
  const Tensor& first = l->params[0];
  const c10::cuda::CUDAGuard guard(first.device());
  const cudaStream_t st = stream_of(first);
  if (lr_at.has_value()) TORCH_CHECK(same_gpu(first, *lr_at) && lr_at->scalar_type() == at::kFloat && lr_at->numel() == 1, "adamw: an fp32 learning rate on the GPU needed");
  struct Batch { bool p16, g16; std::vector<adb200::AdamwTensor> tensors; };
  std::vector<Batch> batches;
  std::vector<Tensor> held;                                  // gradients and parameters that had to be laid out
  std::vector<std::pair<Tensor, Tensor>> back;               // parameters to copy into, from their laid-out copies
  for (size_t i = 0; i < l->params.size(); ++i) {
    const Tensor &p = l->params[i], &g = p.grad();
    const int64_t n = p.numel();
    if (!g.defined() || n == 0) continue;
    TORCH_CHECK(!g.is_sparse(), "adamw: sparse gradients are not supported");
    TORCH_CHECK(same_gpu(first, p) && same_gpu(first, g) && g.sizes() == p.sizes(), "adamw: a gradient does not match its parameter");
    const bool p16 = is_bf16(p, "adamw"), g16 = is_bf16(g, "adamw");
    const void* gp = g.data_ptr();
    void* pp = p.data_ptr();
    if (!g.is_contiguous()) {
      held.push_back(g.contiguous());
      gp = held.back().data_ptr();
    }
    if (!p.is_contiguous()) {
      back.emplace_back(p, p.detach().contiguous());
      pp = back.back().second.data_ptr();
    }
    Batch* b = nullptr;
    for (Batch& c : batches)
      if (c.p16 == p16 && c.g16 == g16 && (int)c.tensors.size() < adb200::kAdamwMost) b = &c;
    if (b == nullptr) {
      batches.push_back({p16, g16, {}});
      b = &batches.back();
      b->tensors.reserve(std::min<size_t>(l->params.size(), adb200::kAdamwMost));
    }
    b->tensors.push_back({pp, gp, n, l->places[i]});
  }
  const bool bits8 = l->m_scale.defined();
  const adb200::AdamwMoments mo{l->m.data_ptr(), l->r.data_ptr(), bits8 ? l->m_scale.data_ptr<float>() : nullptr, bits8 ? l->r_scale.data_ptr<float>() : nullptr};
  adb200::AdamwRule rule{b1, b2, eps, wd, lr_at.has_value() ? lr_at->data_ptr<float>() : nullptr, lr, l->seed,
                         reinterpret_cast<long long*>(l->step.data_ptr<int64_t>()), 0};
  for (size_t k = 0; k < batches.size(); ++k) {
    rule.advance = k + 1 == batches.size();
    launched(adb200::adamw_list_step(batches[k].tensors.data(), (int)batches[k].tensors.size(), batches[k].p16, batches[k].g16, mo, rule, st), "adamw");
  }
  for (auto& b : back) {
    at::NoGradGuard no_grad;
    b.first.detach().copy_(b.second);
  }
  return (int64_t)batches.size();
}

}  // namespace

void register_lm(pybind11::module& m) {
  m.def("rms_norm", &rms_norm);
  m.def("gated_scan", &gated_scan);
  m.def("backward_kernels", &backward_kernels);
  m.def("rms_norm_fwd", &rms_norm_fwd);
  m.def("rms_norm_bwd", &rms_norm_bwd);
  m.def("rms_norm_8bit", &rms_norm_8bit);
  m.def("quantize_rows", &quantize_rows);
  m.def("gemm_8bit", &gemm_8bit, py::arg("codes"), py::arg("scales"), py::arg("weight_codes"), py::arg("weight_scales"), py::arg("bias"), py::arg("error"),
        py::arg("bn") = 0, py::arg("split") = 0);
  m.def("gated_scan_fwd", &gated_scan_fwd);
  m.def("gated_scan_bwd", &gated_scan_bwd);
  pybind11::class_<AdamwList, std::shared_ptr<AdamwList>>(m, "_AdamwList");
  m.def("adamw_list", &adamw_list);
  m.def("adamw_views", &adamw_views);
  m.def("adamw_list_step", &adamw_list_step);
  m.attr("ADAMW_BLOCK") = adb200::kAdamwBlock;
}
