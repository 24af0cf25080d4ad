"""AdamW over a list of tensors against the formula in 64 bits.

fp32 arithmetic adds a few roundings (2^-22 of the sizes that are added); bf16 parameters are rounded to 8 bits. Moments in 8 bits lie within
one step of their e4m3 value, an eighth of the power of two below, and right in the mean."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [1, 2, 3, 255, 256, 257, 300, 511, 1000, 4095, 4096, 4097, 5000, 8192, 12289]
LR, BETAS, EPS, WD = 2e-3, (0.9, 0.999), 1e-8, 0.05


def _params(sizes, dtype, grad_dtype, seed=0, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    params = []
    for n in sizes:
        flat = torch.randn(n + offset, generator=g, device="cuda").to(dtype)
        p = torch.nn.Parameter(flat[offset:])
        grad = (torch.randn(n + offset, generator=g, device="cuda") * 10.0 ** float(torch.randint(-6, 1, (1,), generator=g, device="cuda"))).to(grad_dtype)
        if grad_dtype == dtype:
            p.grad = grad[offset:]
        else:
            p.grad_dtype = None                 # a gradient of another type than its parameter's
            p.grad = grad[offset:]
        params.append(p)
    return params


def _exact(p, g, m, v, t):
    b1, b2 = BETAS
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    move = LR / (1 - b1 ** t) * m / (v.sqrt() / (1 - b2 ** t) ** 0.5 + EPS)
    return p * (1 - LR * WD) - move, m, v, move.abs() + p.abs()


def _slots(opt, p):
    s = opt.slots_of(p)
    return (torch.zeros_like(p, dtype=torch.float64),) * 2 if s is None else (s["exp_avg"].double(), s["exp_avg_sq"].double())


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)]
if hasattr(torch.Tensor, "grad_dtype"):
    TYPES += [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("dtype,grad_dtype", TYPES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_steps(dtype, grad_dtype, bits, offset):
    from autodist_b200.optim import ListAdamW
    params = _params(SIZES, dtype, grad_dtype, offset=offset)
    opt = ListAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=bits)
    for t in range(1, 5):
        for p in params:
            p.grad.mul_(-0.7)
        before = [(p.detach().double(), *_slots(opt, p)) for p in params]
        opt.step()
        for p, (w, m, v) in zip(params, before):
            w, m, v, size = _exact(w, p.grad.double(), m, v, t)
            bound = 2.0 ** -21 * size + (2.0 ** -8 * w.abs() if dtype == torch.bfloat16 else 0)
            assert ((p.detach().double() - w).abs() <= bound).all()
            got_m, got_v = _slots(opt, p)
            if bits == 32:
                assert ((got_m - m).abs() <= 2.0 ** -22 * (m.abs() + p.grad.double().abs())).all() and ((got_v - v).abs() <= 2.0 ** -21 * v).all()
            else:
                for got, want, name in ((got_m, m, "exp_avg"), (got_v.sqrt(), v.sqrt(), "exp_avg_sq")):
                    n = p.numel()
                    scale = opt.state[p][name + "_scale"].double()
                    most = torch.nn.functional.pad(want, (0, -n % 256)).view(-1, 256).abs().amax(1)
                    assert ((scale - most / 448).abs() <= 2.0 ** -20 * (scale + 1e-12)).all()
                    scale = scale.repeat_interleave(256)[:n]
                    ulp = torch.exp2((want.abs() / scale).clamp_min(2.0 ** -6).log2().floor() - 3) * scale
                    assert ((got - want).abs() <= ulp * (1 + 2.0 ** -10)).all()
                    assert ((got != 0) | (want == 0)).all()
        assert opt.slots_of(params[0])["step"] == t


@pytest.mark.parametrize("bits", [8, 32])
def test_the_kernel_is_the_expression(bits):
    """The same step as PyTorch expressions on the host: fp32 results a rounding apart, 8-bit values the same but where a rounding decides."""
    from autodist_b200.optim import ListAdamW
    params = _params(SIZES, torch.float32, torch.float32)
    host = [torch.nn.Parameter(p.detach().cpu()) for p in params]
    for p, h in zip(params, host):
        h.grad = p.grad.cpu()
    opts = [ListAdamW(q, lr=LR, state_bits=bits, seed=5) for q in (params, host)]
    other = 0
    for _ in range(3):
        for o in opts:
            o.step()
        there, here = (o.buffers for o in opts)
        total = 0
        for k in here:
            a, b = there[k].cpu().float(), here[k].float()
            if bits == 8 and not k.endswith("scale"):
                other += int((a != b).sum())
                total += a.numel()
            else:
                assert torch.allclose(a, b, rtol=1e-5, atol=0 if bits == 8 else 1e-12)
        assert other <= 2e-3 * max(total, 1)
        for p, h in zip(params, host):
            assert torch.allclose(p.detach().cpu(), h.detach(), rtol=1e-6, atol=1e-6 if other else 1e-8)
        opts[0].load_buffers(int(opts[0].slots_of(params[0])["step"]), **{k: v.cuda() for k, v in here.items()})


def test_rounding_is_right_in_the_mean_and_repeats():
    from autodist_b200.optim import ListAdamW
    n = 1 << 20
    g = torch.Generator(device="cuda").manual_seed(9)
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = torch.randn(n, generator=g, device="cuda")
    runs = []
    for seed in (1, 1, 2):
        opt = ListAdamW([p], lr=0.0, state_bits=8, seed=seed)
        opt.step()
        runs.append({k: v.clone() for k, v in opt.buffers.items()})
        m, r = (opt.slots_of(p)["exp_avg"].double(), opt.slots_of(p)["exp_avg_sq"].double().sqrt())
        for got, want in ((m, 0.1 * p.grad.double()), (r, 0.001 ** 0.5 * p.grad.double().abs())):
            off = (got - want) / want.abs().mean()
            assert abs(float(off.mean())) < 5 * float(off.std()) / n ** 0.5 + 2.0 ** -17
    for k in runs[0]:
        assert torch.equal(runs[0][k].float(), runs[1][k].float())
    assert not torch.equal(runs[0]["exp_avg"].float(), runs[2]["exp_avg"].float())
    # a second moment far above what the gradients feed it decays as it should: by the root of 0.999 a step, not at all to the nearest
    opt = ListAdamW([p], lr=0.0, state_bits=8)
    opt.step()
    start = opt.slots_of(p)["exp_avg_sq"].sqrt().double().mean()
    p.grad.zero_()
    for _ in range(60):
        opt.step()
    ratio = float(opt.slots_of(p)["exp_avg_sq"].sqrt().double().mean() / start)
    assert abs(ratio - 0.999 ** 30) < 0.004


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors_and_none_without_a_gradient(bits):
    from autodist_b200 import ops
    from autodist_b200.optim import ListAdamW
    sizes = [(37 * k) % 600 + 1 for k in range(1500)]
    params = _params(sizes, torch.float32, torch.float32)
    for k in (0, 7, 800, 1499):
        params[k].grad = None
    before = [p.detach().clone() for p in params]
    opt = ListAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=bits)
    opt.step()
    launched = ops.launch_count
    opt.step()
    assert ops.launch_count - launched == 3 and opt.slots_of(params[0])["step"] == 2
    for k in (0, 7, 800, 1499):
        assert torch.equal(params[k], before[k]) and not opt.slots_of(params[k])["exp_avg"].any()
    m = v = torch.zeros((), dtype=torch.float64, device="cuda")
    for k in (1, 6, 639, 640, 641, 1279, 1281, 1498):
        w, m, v, size = _exact(before[k].double(), params[k].grad.double(), torch.zeros_like(before[k], dtype=torch.float64), 0.0, 1)
        assert not torch.equal(params[k], before[k])
        assert ((params[k].double() - w).abs() <= 2 * LR + 2.0 ** -8 * size).all()       # a step of about the learning rate further


def test_tensors_of_all_types_in_one_step_and_views():
    from autodist_b200.optim import ListAdamW
    a, b = (_params([700, 300], d, d, seed=3) for d in (torch.float32, torch.bfloat16))
    square = torch.nn.Parameter(torch.randn(40, 30, device="cuda").t())             # neither it nor its gradient is dense
    square.grad = torch.randn(30, 80, device="cuda")[:, ::2]
    empty = torch.nn.Parameter(torch.zeros(0, device="cuda"))
    empty.grad = torch.zeros(0, device="cuda")
    params = [a[0], b[0], empty, square, b[1], a[1]]
    before = [p.detach().double() for p in params]
    opt = ListAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=32)
    opt.step()
    assert opt.slots_of(empty)["step"] == 1
    for p, w in zip(params, before):
        w, m, v, size = _exact(w, p.grad.double(), 0.0, 0.0, 1)
        assert ((p.detach().double() - w).abs() <= 2.0 ** -21 * size + (2.0 ** -8 * w.abs() if p.dtype == torch.bfloat16 else 0)).all()
        assert ((opt.slots_of(p)["exp_avg"].double() - m).abs() <= 2.0 ** -21 * m.abs()).all()


def test_groups_rates_on_the_gpu_and_a_storage_that_changes():
    from autodist_b200.optim import ListAdamW
    params = _params([400, 900], torch.float32, torch.float32)
    lr = torch.tensor([LR], device="cuda")
    opt = ListAdamW([{"params": params[:1]}, {"params": params[1:], "weight_decay": 0.5}], lr=lr, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=32)
    before = [p.detach().double() for p in params]
    opt.step()
    w, *_ = _exact(before[0], params[0].grad.double(), 0.0, 0.0, 1)
    assert torch.allclose(params[0].double(), w, rtol=1e-6, atol=1e-6)
    w, *_ = _exact(before[1], params[1].grad.double(), 0.0, 0.0, 1)
    assert torch.allclose(params[1].double(), w - before[1] * LR * (0.5 - WD), rtol=1e-6, atol=1e-6)
    params[0].data = params[0].data.clone()
    before = params[0].detach().clone()
    lr.zero_()
    opt.step()
    assert torch.equal(before, params[0])
    lr.fill_(LR)
    opt.step()
    assert not torch.equal(before, params[0])


def test_captured_in_a_graph():
    from autodist_b200.optim import ListAdamW
    eager, graphed = (_params([300, 5000], torch.float32, torch.float32, seed=4) for _ in range(2))
    opts = [ListAdamW(q, lr=LR, state_bits=8) for q in (eager, graphed)]
    for o in opts:
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[1].step()
    for _ in range(3):
        opts[0].step()
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(eager, graphed))
    assert opts[1].slots_of(graphed[0])["step"] == 4


def test_moments_that_are_zero_tiny_or_not_finite():
    from autodist_b200.optim import ListAdamW
    p = torch.nn.Parameter(torch.ones(256 * 4, device="cuda"))
    p.grad = torch.randn(256 * 4, device="cuda")
    p.grad[:256] = 0
    p.grad[256:512] = 1e-33
    p.grad[512] = float("nan")
    opt = ListAdamW([p], lr=LR, weight_decay=0.0, state_bits=8)
    opt.step()
    assert (p[:256] == 1).all() and p[256:512].isfinite().all() and p[512].isnan() and p[513:].isfinite().all()
    opt.step()
    assert (p[:256] == 1).all() and p[256:512].isfinite().all() and p[512:768].isnan().all() and p[768:].isfinite().all()


@pytest.mark.parametrize("bits", [8, 32])
def test_states_are_saved_and_restored(bits):
    from autodist_b200.optim import ListAdamW
    params = _params([300, 5000], torch.float32, torch.float32)
    opt = ListAdamW(params, lr=LR, state_bits=bits, seed=3)
    opt.step()
    saved, values = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in params]
    opt.step()
    after = [p.detach().clone() for p in params]
    again = ListAdamW(params, lr=1.0, state_bits=bits, seed=3)
    again.load_state_dict(saved)
    with torch.no_grad():
        for p, v in zip(params, values):
            p.copy_(v)
    again.step()
    assert all(torch.equal(p, a) for p, a in zip(params, after))
    assert all(torch.equal(again.buffers[k].float(), opt.buffers[k].float()) for k in opt.buffers)
    # as fp32 slots, under torch.optim's names: what 32 bits hold comes back, what 8 bits hold is rounded once more at most
    third = ListAdamW(params, lr=LR, state_bits=bits)
    for p in params:
        third.load_slots(p, opt.slots_of(p), opt.slots_of(p)["step"])
    for p in params:
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.allclose(third.slots_of(p)[k], opt.slots_of(p)[k], rtol=1e-5, atol=0)
        assert third.slots_of(p)["step"] == 2
    with pytest.raises(ValueError, match="bits"):
        ListAdamW(params, state_bits=40 - bits).load_state_dict(saved)
    with pytest.raises(ValueError, match="other parameter groups"):
        ListAdamW(params[:1], state_bits=bits).load_state_dict(saved)


def test_places_past_31_bits():
    from autodist_b200.optim import ListAdamW
    n = 2 ** 31 + 5000
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    p.grad[-3000:] = torch.randn(3000, device="cuda").bfloat16()
    p.grad[:100] = 1.0
    opt = ListAdamW([p], lr=LR, weight_decay=0.0, state_bits=8)
    opt.step()
    assert torch.allclose(p[-3000:].float(), -LR * p.grad[-3000:].float().sign(), rtol=2.0 ** -7) and (p[:100] < 0).all()
    assert not p[100:2 ** 20].any() and not p[-3100:-3000].any()


def test_refusals():
    from autodist_b200.optim import ListAdamW
    p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    for bad, what in (({"state_bits": 16}, "8 or in 32"), ({"lr": -1.0}, "learning rate"), ({"betas": (1.0, 0.9)}, "betas"), ({"eps": -1.0}, "eps"),
                      ({"weight_decay": -0.1}, "weight decay")):
        with pytest.raises(ValueError, match=what):
            ListAdamW([p], **bad)
    half = torch.nn.Parameter(torch.zeros(10, device="cuda", dtype=torch.float16))
    half.grad = torch.zeros_like(half)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ListAdamW([half]).step()
    host = torch.nn.Parameter(torch.zeros(10))
    with pytest.raises(ValueError, match="one device"):
        ListAdamW([p, host]).step()
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]], device="cuda"), torch.ones(1, device="cuda"), (10,))
    with pytest.raises(RuntimeError, match="sparse"):
        ListAdamW([p]).step()
    p.grad = None
    opt = ListAdamW([p], lr=torch.tensor([1e-3, 1e-3], device="cuda"))
    p.grad = torch.zeros(10, device="cuda")
    with pytest.raises(RuntimeError, match="learning rate"):
        opt.step()
    with pytest.raises(ValueError, match="needed"):
        opt.load_buffers(1, exp_avg=torch.zeros(256, device="cuda"))
    with pytest.raises(ValueError, match="several groups"):
        ListAdamW([{"params": [p]}, {"params": [host]}]).buffers
