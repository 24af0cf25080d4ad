"""The recurrent language model's operators on the host: the plain expressions that CPU tensors, second derivatives and transforms go through."""
import os
import re

import pytest
import torch

from autodist_b200.ops import functional as F
from autodist_b200.optim import ListAdamW

BINDINGS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "autodist_b200", "csrc", "lm_bindings.cpp")


def test_norm():
    x, w, r = torch.randn(3, 5, 24), torch.rand(24) + 0.5, torch.randn(3, 5, 24)
    y, s = F.rms_norm(x, w, r, 1e-5)
    want = (x + r).double()
    want = want / (want.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
    assert torch.equal(s, x + r) and torch.allclose(y.double(), want, rtol=1e-5, atol=1e-6)
    assert F.rms_norm(x.bfloat16(), w).dtype == torch.bfloat16
    codes, scales, s = F.rms_norm_8bit(x, w, r, 1e-5)
    held = codes.double() * scales.double()[..., None]
    assert ((held - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * scales[..., None] + 1e-6).all()
    assert torch.autograd.gradcheck(lambda a: F.rms_norm(a, w[:4].clone())[0].double(), torch.randn(2, 4, requires_grad=True), eps=1e-2, atol=1e-2)


@pytest.mark.parametrize("gate", [False, True])
def test_recurrence(gate):
    x, f, i = (torch.randn(2, 9, 6, requires_grad=True) for _ in range(3))
    state, reset = torch.randn(2, 6, requires_grad=True), torch.zeros(2, 9, dtype=torch.bool)
    reset[1, 4] = True
    y, last = F.gated_recurrence(x, f, i if gate else None, state, reset, 0.5)
    h = state.double()
    for t in range(9):
        a = torch.sigmoid(f[:, t].double() + 0.5)
        u = torch.sigmoid(i[:, t].double()) if gate else 1 - a
        h = torch.where(reset[:, t, None], torch.zeros_like(h), a * h) + u * x[:, t].double()
        assert torch.allclose(y[:, t].double(), h, atol=1e-5)
    assert torch.allclose(last.double(), h, atol=1e-5)
    (y.sum() + last.sum()).backward()
    assert all(t.grad.isfinite().all() for t in (x, f, state)) and (i.grad is not None) == gate
    empty, kept = F.gated_recurrence(x[:, :0], f[:, :0], state=state)
    assert empty.shape == (2, 0, 6) and torch.equal(kept, state)


def test_vmap_goes_through_the_expression():
    x, f = torch.randn(4, 2, 5, 3), torch.randn(4, 2, 5, 3)
    y, _ = torch.func.vmap(F.gated_recurrence)(x, f)
    assert torch.allclose(y[1], F.gated_recurrence(x[1], f[1])[0], atol=1e-6)
    w = torch.rand(3)
    assert torch.allclose(torch.func.vmap(lambda a: F.rms_norm(a, w))(x), F.rms_norm(x, w), atol=1e-6)


def test_product_in_8_bits():
    x, w, b = torch.randn(2, 3, 40), torch.randn(7, 40), torch.randn(7)
    q, s = F.quantize_rows(x)
    qw, sw = F.quantize_rows(w)
    y = F.linear_8bit(q, s, qw, sw, b)
    want = (q.double() * s.double()[..., None]) @ (qw.double() * sw.double()[:, None]).t() + b
    assert y.dtype == torch.bfloat16 and torch.allclose(y.double(), want, rtol=2.0 ** -8, atol=1e-4)
    with pytest.raises(ValueError, match="do not match"):
        F.linear_8bit(q, s, qw[:, :39], sw)
    with pytest.raises(RuntimeError, match="no gradient"):
        F.quantize_rows(x.requires_grad_(True))


def _trained(make, steps=60):
    torch.manual_seed(3)
    params = [torch.nn.Parameter(torch.randn(n)) for n in (5, 300, 1031)]
    opt = make(params)
    for _ in range(steps):
        for p in params:
            p.grad = torch.randn(p.shape) + 0.3 * p.detach()
        opt.step()
    return opt, params


def test_adamw_in_32_bits_is_the_librarys():
    _, own = _trained(lambda ps: ListAdamW(ps, lr=1e-2, weight_decay=0.1, state_bits=32))
    _, library = _trained(lambda ps: torch.optim.AdamW(ps, lr=1e-2, weight_decay=0.1))
    for a, b in zip(own, library):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


def test_adamw_in_8_bits_follows_it():
    opt, own = _trained(lambda ps: ListAdamW(ps, lr=1e-2, state_bits=8))
    _, library = _trained(lambda ps: torch.optim.AdamW(ps, lr=1e-2))
    for a, b in zip(own, library):
        assert float((a - b).norm() / b.norm()) < 0.03
    assert opt.buffers["exp_avg"].dtype == torch.float8_e4m3fn and opt.slots_of(own[0])["step"] == 60
    held = sum(b.numel() * b.element_size() for b in opt.buffers.values())
    assert held == (256 + 512 + 1280) * 2 + 8 * 8


def test_adamw_refusals_and_states():
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(ValueError, match="8 or in 32"):
        ListAdamW([p], state_bits=4)
    with pytest.raises(ValueError, match="learning rate"):
        ListAdamW([p], lr=-1.0)
    opt = ListAdamW([p])
    assert opt.slots_of(p) is None
    opt.step()                                      # no gradient: nothing happens
    assert opt.slots_of(p)["step"] == 0 and not p.any()
    opt, params = _trained(lambda ps: ListAdamW(ps, seed=4), 3)
    again = ListAdamW(params, seed=4)
    again.load_state_dict(opt.state_dict())
    assert all(torch.equal(again.buffers[k].float(), opt.buffers[k].float()) for k in opt.buffers)


@pytest.mark.parametrize("name", ["rms_norm_fwd", "rms_norm_bwd", "rows_8bit", "gemm_8bit", "gated_scan_fwd", "gated_scan_bwd", "adamw_list_step"])
def test_the_device_is_switched_before_the_stream_is_asked_for(name):
    with open(BINDINGS) as f:
        source = f.read()
    body = re.search(r"^\S[^\n]*\b%s\((?:[^{]|\n)*?\{\n(.*?)^\}" % name, source, re.M | re.S).group(1)
    assert 0 <= body.find("c10::cuda::CUDAGuard guard(") < body.find("stream_of(")
