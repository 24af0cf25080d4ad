"""Root-mean-square norm against the formula in 64 bits.

Tolerances: bf16 rounds to 8 bits (an error of 2^-8 of the value at most), e4m3 to 4 bits (2^-4, or half of its smallest step of 2^-9 scales);
sums of fp32 values are a chain of at most some 60 additions here, 2^-18 of the sum of the sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SUMS = 2.0 ** -18
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -22}
EPS = 1e-5


def _inputs(rows, width, dtype, weight_dtype=torch.float32, residual=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + width)
    x, res, dy, ds = (torch.randn(rows, width, generator=g, device="cuda").mul_(s).to(dtype) for s in (1.0, 3.0, 1.0, 0.5))
    w = (torch.randn(width, generator=g, device="cuda") * 0.2 + 1).to(weight_dtype)
    return x, w, res if residual else None, dy, ds if residual else None


def _reference(x, w, res, eps=EPS):
    s = x if res is None else (x.float() + res.float()).to(x.dtype)
    d = s.double()
    rstd = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    return s, d * rstd, rstd, d * rstd * w.double()


def _near(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want.double()).abs() - bound
    assert not torch.isnan(off).any() and (off <= 0).all(), float(off.max())


WIDTHS = [1, 2, 3, 7, 8, 31, 32, 33, 64, 100, 255, 256, 257, 512, 1000, 1001, 1024, 2047, 2048, 4096, 4104, 8191, 8192, 12290]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,weight_dtype", [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_and_gradients(width, dtype, weight_dtype, residual):
    from autodist_b200.ops import functional as F
    for rows in (1, 5, 67):
        x, w, res, dy, ds = _inputs(rows, width, dtype, weight_dtype, residual)
        s, n, rstd, y = _reference(x, w, res)
        with torch.no_grad():
            free = F.rms_norm(x, w, res, EPS)
        leaves = [t.requires_grad_(True) for t in (x, w, res) if t is not None]
        out = F.rms_norm(x, w, res, EPS)
        for a, b in zip(out if residual else (out,), free if residual else (free,)):
            assert torch.equal(a, b)                    # the same with and without a gradient
        got_y = out[0] if residual else out
        _near(got_y, y, (ROUND[dtype] + SUMS) * y.abs())
        if residual:
            assert torch.equal(out[1], s)
        grads = torch.autograd.grad(out, leaves, (dy, ds) if residual else dy)
        g = dy.double() * w.double()
        along = (g * n).mean(-1, keepdim=True)
        dx = rstd * (g - n * along) + (ds.double() if residual else 0)
        sizes = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)) + (ds.double().abs() if residual else 0)
        _near(grads[0], dx, ROUND[dtype] * dx.abs() + 2 * SUMS * sizes)
        if residual:
            assert torch.equal(grads[2], grads[0])
        dw = (dy.double() * n).sum(0)
        _near(grads[1], dw, ROUND[weight_dtype] * dw.abs() + 2 * SUMS * (dy.double() * n).abs().sum(0))


@pytest.mark.parametrize("rows", [300, 2049, 5000])
@pytest.mark.parametrize("width", [40, 768, 1024, 3001])
def test_gradient_of_a_shared_weight_over_many_rows(rows, width):
    from autodist_b200.ops import functional as F
    x, w, _, dy, _ = _inputs(rows, width, torch.bfloat16, residual=False)
    _, n, _, _ = _reference(x, w, None)
    w.requires_grad_(True)
    first = torch.autograd.grad(F.rms_norm(x, w, eps=EPS), w, dy)[0]
    sizes = (dy.double() * n).abs().sum(0)
    _near(first, (dy.double() * n).sum(0), 2 * SUMS * sizes)
    assert torch.equal(first, torch.autograd.grad(F.rms_norm(x, w, eps=EPS), w, dy)[0])       # the order of the sums is fixed


@pytest.mark.parametrize("width", [159, 161, 519, 520, 1025, 1301, 2047, 2560, 4095, 5001, 8185, 8191])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows_with_groups_of_any_number_of_warps(width, dtype):
    from autodist_b200.ops import functional as F
    x, w, res, dy, ds = _inputs(1203, width, dtype)
    s, n, rstd, y = _reference(x, w, res)
    codes, scales, total = F.rms_norm_8bit(x, w, res, EPS)
    assert torch.equal(total, s)
    most = y.abs().amax(1, keepdim=True)
    step = most / 448
    _near(scales.reshape(-1, 1), step, 2 * SUMS * step)
    _near(codes.double() * scales.double().reshape(-1, 1), y, (2.0 ** -4 + 4 * SUMS) * y.abs() + step * 2.0 ** -10)
    leaves = [t.requires_grad_(True) for t in (x, w, res)]
    out = F.rms_norm(x, w, res, EPS)
    _near(out[0], y, (ROUND[dtype] + SUMS) * y.abs())
    grads = torch.autograd.grad(out, leaves, (dy, ds))
    g = dy.double() * w.double()
    dx = rstd * (g - n * (g * n).mean(-1, keepdim=True)) + ds.double()
    sizes = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)) + ds.double().abs()
    _near(grads[0], dx, ROUND[dtype] * dx.abs() + 2 * SUMS * sizes)
    dw = (dy.double() * n).sum(0)
    _near(grads[1], dw, ROUND[torch.float32] * dw.abs() + 2 * SUMS * (dy.double() * n).abs().sum(0))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_output_in_8_bits(width, dtype):
    from autodist_b200.ops import functional as F
    for rows, residual in ((1, True), (70, False), (67, True)):
        x, w, res, _, _ = _inputs(rows, width, dtype, residual=residual)
        s, _, _, y = _reference(x, w, res)
        out = F.rms_norm_8bit(x, w, res, EPS)
        codes, scales = out[:2]
        assert codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32 and codes.shape == x.shape and scales.shape == x.shape[:-1]
        assert codes.data_ptr() % 16 == 0 and (rows == 1 or codes.stride(0) % 16 == 0)
        if residual:
            assert torch.equal(out[2], s)
        most = y.abs().amax(-1)
        _near(scales, most / 448, 2 * SUMS * most / 448)
        _near(codes.double() * scales.double()[:, None], y, 2.0 ** -4 * (1 + 2.0 ** -10) * y.abs() + 2.0 ** -10 * scales.double()[:, None])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 17), (2, 5, 48), (129, 2048), (9, 5001)])
def test_rows_in_8_bits(dtype, shape):
    from autodist_b200.ops import functional as F
    x = torch.randn(*shape, device="cuda").to(dtype)
    x[0] = 0
    codes, scales = F.quantize_rows(x)
    assert codes.shape == x.shape and scales.shape == x.shape[:-1]
    _near(scales, x.double().abs().amax(-1) / 448, 2.0 ** -22 * scales.double())
    _near(codes.double() * scales.double()[..., None], x.double(), 2.0 ** -4 * (1 + 2.0 ** -10) * x.double().abs() + 2.0 ** -10 * scales.double()[..., None])
    assert (scales[0] == 0).all() and (codes[0].float() == 0).all()


@pytest.mark.parametrize("width", [24, 1001, 2048])
def test_rows_that_are_not_finite_or_zero(width):
    from autodist_b200.ops import functional as F
    x, w, _, dy, _ = _inputs(6, width, torch.bfloat16, residual=False)
    clean = F.rms_norm(x, w, eps=EPS)
    codes, scales = F.rms_norm_8bit(x, w, eps=EPS)
    bad = x.clone()
    bad[1] = 0
    bad[2, width // 2] = float("nan")
    bad[4, 0] = float("inf")
    y = F.rms_norm(bad, w, eps=EPS)
    assert (y[1] == 0).all() and y[2].isnan().all()
    assert y[4, 0].isnan() and (y[4, 1:] == 0).all()             # finite over infinity, infinity times zero
    bad_codes, bad_scales = F.rms_norm_8bit(bad, w, eps=EPS)
    assert bad_scales[1] == 0 and (bad_codes[1].float() == 0).all()
    assert bad_scales[2].isnan() and bad_codes[2].float().isnan().all() and bad_scales[4].isnan()
    for i in (0, 3, 5):                                            # the rows beside them
        assert torch.equal(y[i], clean[i]) and torch.equal(bad_codes[i].view(torch.uint8), codes[i].view(torch.uint8)) and bad_scales[i] == scales[i]
    zero = torch.zeros(3, width, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(F.rms_norm(zero, w, eps=EPS), zero, torch.ones(3, width, device="cuda"))
    _near(dx, (w.double() / EPS ** 0.5).expand(3, width), 2.0 ** -18 / EPS ** 0.5 * w.double().abs())


def test_strides_bases_and_orders():
    from autodist_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(5)
    base = torch.randn(64, 3000, generator=g, device="cuda").bfloat16()
    w = torch.randn(500, generator=g, device="cuda")
    views = [base[:, 7:507], base[::3, 8:508], base[:, 16:516].unflatten(0, (4, 16)), base[:500, :].t().contiguous()[:500, :].t(), base[:1, 3:503].expand(9, 500),
             base[:, 0:1000:2]]
    for v in views:
        dense = v.contiguous()
        r = dense * 2
        assert torch.equal(F.rms_norm(v, w), F.rms_norm(dense, w))
        for a, b in zip(F.rms_norm(v, w, r) + F.rms_norm(r, w, v), F.rms_norm(dense, w, r) + F.rms_norm(r, w, dense)):
            assert torch.equal(a, b)
        for a, b in zip(F.rms_norm_8bit(v, w, r), F.rms_norm_8bit(dense, w, r)):
            assert torch.equal(a.float(), b.float())
        leaf, same = v.detach().requires_grad_(True), dense.detach().clone().requires_grad_(True)
        dy = torch.randn(*v.shape, 2, generator=g, device="cuda").bfloat16()[..., 0]
        weight, weight2 = w.clone().requires_grad_(True), w.clone().requires_grad_(True)
        for a, b in zip(torch.autograd.grad(F.rms_norm(leaf, weight), (leaf, weight), dy), torch.autograd.grad(F.rms_norm(same, weight2), (same, weight2), dy.contiguous())):
            assert torch.equal(a, b)
    x = base[:, :500].float().requires_grad_(True)
    dx, = torch.autograd.grad(F.rms_norm(x, w).sum(), x)             # an expanded gradient
    dense, = torch.autograd.grad(F.rms_norm(x, w), x, torch.ones_like(x))
    assert torch.equal(dx, dense)


def test_no_rows():
    from autodist_b200.ops import functional as F
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    y, s = F.rms_norm(x, w, torch.zeros_like(x))
    dx, dw = torch.autograd.grad((y, s), (x, w), (y, s))
    assert y.shape == s.shape == dx.shape == (0, 16) and (dw == 0).all()
    codes, scales = F.rms_norm_8bit(torch.zeros(2, 0, 16, device="cuda"), w.detach())
    assert codes.shape == (2, 0, 16) and scales.shape == (2, 0)


def test_only_some_gradients_are_wanted_or_given():
    from autodist_b200.ops import functional as F
    x, w, res, dy, ds = _inputs(9, 96, torch.float32)
    x.requires_grad_(True)
    y, s = F.rms_norm(x, w, res)
    assert torch.equal(torch.autograd.grad(s, x, ds, retain_graph=True)[0], ds)
    only_y, = torch.autograd.grad(y, x, dy, retain_graph=True)
    both, = torch.autograd.grad((y, s), x, (dy, ds))
    _near(both, only_y.double() + ds.double(), 2.0 ** -20 * (only_y.double().abs() + ds.double().abs()))
    w2 = w.clone().requires_grad_(True)
    dw, = torch.autograd.grad(F.rms_norm(x.detach(), w2, res)[0], w2, dy)
    assert dw.shape == w.shape


def test_against_differences_and_second_derivatives():
    from autodist_b200.ops import functional as F
    x, w, res, dy, ds = _inputs(4, 33, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(1)
    for t in (x, w, res):
        t.requires_grad_(True)
    grads = torch.autograd.grad(F.rms_norm(x, w, res, EPS), (x, w, res), (dy, ds))
    steps = [torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64) for t in (x, w, res)]

    def value(h):
        xs, ws, rs = (t.detach().double() + h * d for t, d in zip((x, w, res), steps))
        s = xs + rs
        return float((s * (s.square().mean(-1, keepdim=True) + EPS).rsqrt() * ws * dy.double()).sum() + (s * ds.double()).sum())
    slope = (value(1e-5) - value(-1e-5)) / 2e-5
    sizes = sum(float((a.double() * d).abs().sum()) for a, d in zip(grads, steps))
    assert abs(sum(float((a.double() * d).sum()) for a, d in zip(grads, steps)) - slope) <= 1e-5 * sizes
    # a gradient of a gradient, against the same of the plain expression on the host
    def twice(*leaves):
        y, s = F.rms_norm(*leaves, EPS)
        first = torch.autograd.grad((y * y).sum() + s.sum(), leaves, create_graph=True)
        return torch.autograd.grad(sum((f * f).sum() for f in first), leaves)
    there = twice(*(t.detach().clone().requires_grad_(True) for t in (x, w, res)))
    here = twice(*(t.detach().cpu().requires_grad_(True) for t in (x, w, res)))
    for a, b in zip(there, here):
        assert torch.allclose(a.cpu(), b, rtol=1e-3, atol=1e-3 * float(b.abs().max()))


def test_on_another_stream():
    from autodist_b200.ops import functional as F
    x, w, res, _, _ = _inputs(513, 1024, torch.bfloat16)
    want = F.rms_norm(x, w, res)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.rms_norm(x, w, res)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_31_bits():
    from autodist_b200.ops import functional as F
    rows, width = 2 ** 19 + 3, 4104
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(width, device="cuda")
    x[-3:] = torch.randn(3, width, device="cuda").bfloat16()
    y = F.rms_norm(x, w)
    assert torch.equal(y[-3:], F.rms_norm(x[-3:], w)) and not y[:1000].any()
    del y
    codes, scales = F.rms_norm_8bit(x, w)
    few = F.rms_norm_8bit(x[-3:], w)
    assert torch.equal(codes[-3:].float(), few[0].float()) and torch.equal(scales[-3:], few[1])
    leaf = x.requires_grad_(True)
    y = F.rms_norm(leaf, w)
    dx, = torch.autograd.grad(y, leaf, y.detach())
    part = x[-3:].detach().requires_grad_(True)
    y = F.rms_norm(part, w)
    assert torch.equal(dx[-3:], torch.autograd.grad(y, part, y.detach())[0])


def test_refusals():
    from autodist_b200 import ops
    from autodist_b200.ops import functional as F
    x, w = torch.ones(2, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (x.half(), x.double(), x.int()):
        with pytest.raises(TypeError, match="bf16 or fp32"):
            F.rms_norm(bad, w)
    with pytest.raises(ValueError, match="weight for each column"):
        F.rms_norm(x, w[:7])
    with pytest.raises(TypeError, match="weight must be"):
        F.rms_norm(x, w.bfloat16())
    with pytest.raises(ValueError, match="residual"):
        F.rms_norm(x, w, x.bfloat16())
    with pytest.raises(ValueError, match="residual"):
        F.rms_norm(x, w, x[:1])
    with pytest.raises(ValueError, match="at least one element"):
        F.rms_norm(x[:, :0], w[:0])
    with pytest.raises(RuntimeError, match="GPU"):
        F.rms_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match="GPU"):
        F.rms_norm(x, w, x.cpu())
    with pytest.raises(RuntimeError, match="no gradient"):
        F.rms_norm_8bit(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError, match="no gradient"):
        F.quantize_rows(x)
    E = ops.ext(required=True)
    with pytest.raises(RuntimeError, match="GPU"):
        E.rms_norm_fwd(x.detach().cpu(), w, None, 1e-6)
    with pytest.raises(RuntimeError, match="gradient"):
        E.rms_norm_bwd(x.detach()[:1], None, x.detach(), w, 1e-6)
