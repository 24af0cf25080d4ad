"""Operators of a gated recurrent language model: root-mean-square norm (with the residual's addition; with an output in 8 bits), a gated
linear recurrence over time, and the product of 8-bit rows.

CUDA tensors run on the hand-written kernels, CPU tensors on the plain PyTorch expressions below, which are also what second
derivatives, forward-mode derivatives and ``torch.func`` transforms go through.
"""
import math

import torch
import torch.nn.functional as F

from autodist_b200 import ops

#: Largest e4m3 value: a row in 8 bits is scaled so that its largest element has this size.
E4M3_MAX = 448.0

_STREAM_TYPES = (torch.bfloat16, torch.float32)


def _kernels(x):
    """Whether the kernels compute this: tensors on a GPU, and no transform but reverse-mode differentiation going on."""
    return x.is_cuda and not torch._C._are_functorch_transforms_active() and torch.autograd.forward_ad._current_level < 0


def _wants_gradient(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _differentiated_again(plain, inputs, grads_of_outputs):
    """Gradients of ``plain(*inputs)`` that can be differentiated themselves (``create_graph``); ``None`` for inputs that need none."""
    wanted = [t is not None and t.requires_grad for t in inputs]
    # aliases: what is being differentiated may be an output of the very node that asks, which the engine has locked
    inputs = [t.view_as(t) if w else t for t, w in zip(inputs, wanted)]
    outs, grads = zip(*((o, g) for o, g in zip(plain(*inputs), grads_of_outputs) if g is not None))
    found = iter(torch.autograd.grad(outs, [t for t, w in zip(inputs, wanted) if w], grads, create_graph=True, allow_unused=True))
    return [next(found) if w else None for w in wanted]


# ---------------------------------------------------------------------------------------------------------------- norm
def _check_norm(name, x, weight, residual):
    if x.dtype not in _STREAM_TYPES:
        raise TypeError(f"{name}: bf16 or fp32 needed, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name}: rows of at least one element needed, got {tuple(x.shape)}")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"{name}: a weight for each column needed, got {tuple(weight.shape)} for {tuple(x.shape)}")
    if weight.dtype not in (torch.float32, x.dtype):
        raise TypeError(f"{name}: the weight must be fp32 or of the input's type, got {weight.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{name}: the residual must have the input's shape and type, got {tuple(residual.shape)} {residual.dtype}")


def _norm_plain(x, weight, residual, eps):
    s = x if residual is None else x + residual
    f = s.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps) * weight.float()
    return y, s


def _norm_again(s, weight, eps, dy, ds):
    """Gradients of what was normed and of the weight, for ``create_graph``."""
    return _differentiated_again(lambda t, w: (_norm_plain(t, w, None, eps)[0].to(t.dtype), t), (s, weight), (dy, ds))


def rms_norm(x, weight, residual=None, eps=1e-6):
    """``s * rsqrt(mean(s^2) + eps) * weight`` over the last dimension, with ``s = x``, or ``s = x + residual`` rounded to their type; then
    ``(norm, s)`` is returned. bf16 or fp32; the weight in fp32 or in the input's type. Sums are fp32."""
    if not _kernels(x):
        _check_norm("rms_norm", x, weight, residual)
        y, s = _norm_plain(x, weight, residual, eps)
        return y.to(x.dtype) if residual is None else (y.to(x.dtype), s)
    try:
        y, s = ops.ext(required=True).rms_norm(x, weight, residual, eps)
    except RuntimeError:                        # the binding checks all of this too; here the argument at fault is named
        _check_norm("rms_norm", x, weight, residual)
        raise
    return y if residual is None else (y, s)


def _no_gradient(name, *tensors):
    if _wants_gradient(*tensors):
        raise RuntimeError(f"{name}: rows in 8 bits carry no gradient; call it under torch.no_grad()")


def _codes_plain(y):
    scale = y.abs().amax(-1) / E4M3_MAX
    held = torch.where(scale[..., None] == 0, torch.zeros_like(y), y / scale[..., None])
    return held.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def rms_norm_8bit(x, weight, residual=None, eps=1e-6):
    """``rms_norm`` with its output in 8 bits: ``(codes, scales)``, or ``(codes, scales, s)`` with a residual. ``codes`` (``float8_e4m3fn``)
    times its row's fp32 scale is the norm's output, the row's largest element being 448 scales; rows of zeros have the scale 0. Rows of
    ``codes`` start on 16-byte boundaries, as ``linear_8bit`` reads them. Not differentiable."""
    _no_gradient("rms_norm_8bit", x, weight, residual)
    if not _kernels(x):
        _check_norm("rms_norm_8bit", x, weight, residual)
        y, s = _norm_plain(x, weight, residual, eps)
        return _codes_plain(y) if residual is None else _codes_plain(y) + (s,)
    try:
        codes, scales, s = ops.ext(required=True).rms_norm_8bit(x, weight, residual, eps)
    except RuntimeError:
        _check_norm("rms_norm_8bit", x, weight, residual)
        raise
    return (codes, scales) if residual is None else (codes, scales, s)


def quantize_rows(x):
    """``(codes, scales)`` of the rows of ``x`` (bf16 or fp32, last dimension) as ``rms_norm_8bit`` returns them: for weights, once, and for
    activations that no norm produces. Not differentiable: a trained weight is passed detached."""
    if x.dtype not in _STREAM_TYPES:
        raise TypeError(f"quantize_rows: bf16 or fp32 needed, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize_rows: rows of at least one element needed, got {tuple(x.shape)}")
    _no_gradient("quantize_rows", x)
    return ops.ext(required=True).quantize_rows(x) if _kernels(x) else _codes_plain(x.float())


# ---------------------------------------------------------------------------------------------------------------- product in 8 bits
def _check_linear(codes, scales, weight_codes, weight_scales, bias):
    if codes.dtype != torch.float8_e4m3fn or weight_codes.dtype != torch.float8_e4m3fn:
        raise TypeError(f"linear_8bit: float8_e4m3fn rows and weight needed, got {codes.dtype} and {weight_codes.dtype}")
    if codes.dim() < 1 or weight_codes.dim() != 2 or codes.shape[-1] != weight_codes.shape[1] or codes.shape[-1] < 1:
        raise ValueError(f"linear_8bit: rows of {tuple(codes.shape)} and a weight of {tuple(weight_codes.shape)} do not match")
    if scales.dtype != torch.float32 or scales.shape != codes.shape[:-1] or weight_scales.dtype != torch.float32 or \
            weight_scales.shape != weight_codes.shape[:1]:
        raise ValueError("linear_8bit: an fp32 scale for each row of both sides needed")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != weight_scales.shape):
        raise ValueError("linear_8bit: an fp32 bias for each output needed")


def linear_8bit(codes, scales, weight_codes, weight_scales, bias=None):
    """``(codes * scales) @ (weight_codes * weight_scales).T + bias`` in bf16 for rows ``[..., K]`` and a weight ``[N, K]`` of
    ``float8_e4m3fn`` with an fp32 scale each (``rms_norm_8bit``, ``quantize_rows``). Products are exact, sums fp32. Not differentiable."""
    _no_gradient("linear_8bit", scales, weight_scales, bias)
    if codes.is_cuda:
        from autodist_b200.ops.functional import _error_flag
        try:
            return ops.ext(required=True).gemm_8bit(codes, scales, weight_codes, weight_scales, bias, _error_flag(codes.device))
        except RuntimeError:
            _check_linear(codes, scales, weight_codes, weight_scales, bias)
            raise
    _check_linear(codes, scales, weight_codes, weight_scales, bias)
    y = F.linear(codes.float(), weight_codes.float()) * scales[..., None] * weight_scales
    return (y if bias is None else y + bias).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------------- recurrence
def _scan_plain(x, forget, input_gate, state, reset, forget_bias):
    f = torch.sigmoid(forget.float() + forget_bias)
    u = torch.sigmoid(-(forget.float() + forget_bias)) if input_gate is None else torch.sigmoid(input_gate.float())
    v = u * x.float()
    h = x.new_zeros(x.shape[0], x.shape[2], dtype=torch.float32) if state is None else state
    outs = []
    for t in range(x.shape[1]):
        held = f[:, t] * h
        if reset is not None:
            held = torch.where(reset[:, t, None], torch.zeros_like(held), held)
        h = held + v[:, t]
        outs.append(h)
    y = torch.stack(outs, 1).to(x.dtype) if outs else torch.empty_like(x)
    return y, h if outs or state is None else h.clone()


def _scan_again(x, forget, input_gate, state, reset, forget_bias, dy, dlast):
    """Gradients of the first four, for ``create_graph``."""
    return _differentiated_again(lambda *a: _scan_plain(*a, reset, forget_bias), (x, forget, input_gate, state), (dy, dlast))


def _check_scan(x, forget, input_gate, state, reset):
    if x.dtype not in _STREAM_TYPES:
        raise TypeError(f"gated_recurrence: bf16 or fp32 needed, got {x.dtype}")
    if x.dim() != 3:
        raise ValueError(f"gated_recurrence: [batch, steps, channels] needed, got {tuple(x.shape)}")
    for t, what in ((forget, "forget gate"), (input_gate, "input gate")):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError(f"gated_recurrence: the {what} must have the input's shape and type, got {tuple(t.shape)} {t.dtype}")
    if state is not None and (state.dtype != torch.float32 or state.shape != (x.shape[0], x.shape[2])):
        raise ValueError(f"gated_recurrence: an fp32 state [batch, channels] needed, got {tuple(state.shape)} {state.dtype}")
    if reset is not None and (reset.dtype != torch.bool or reset.shape != x.shape[:2]):
        raise ValueError(f"gated_recurrence: a bool reset [batch, steps] needed, got {tuple(reset.shape)} {reset.dtype}")


def gated_recurrence(x, forget, input_gate=None, state=None, reset=None, forget_bias=0.0):
    """``h_t = f_t * h_{t-1} + u_t * x_t`` channel by channel over ``[batch, steps, channels]``: ``(h in x's type, last state in fp32)``.

    ``f = sigmoid(forget + forget_bias)``; ``u = sigmoid(input_gate)``, or ``1 - f`` without one. ``state``: fp32 ``[batch, channels]``, the
    state in front of the first step (zeros without one); pass the last state on to continue, one token at a time if need be.
    ``reset``: bool ``[batch, steps]``, the steps that forget the state in front of them (a document begins). bf16 or fp32; strided views,
    such as slices of one projection, are read in place. States are fp32 throughout; the backward pass computes them again."""
    if not math.isfinite(forget_bias):
        raise ValueError(f"gated_recurrence: a finite forget_bias needed, got {forget_bias}")
    if not _kernels(x):
        _check_scan(x, forget, input_gate, state, reset)
        return _scan_plain(x, forget, input_gate, state, reset, forget_bias)
    try:
        y, last, _ = ops.ext(required=True).gated_scan(x, forget, input_gate, state, reset, forget_bias)
    except RuntimeError:
        _check_scan(x, forget, input_gate, state, reset)
        raise
    return y, last
