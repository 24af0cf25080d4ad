"""The product of 8-bit rows against the same values multiplied in 64 bits.

e4m3 products are exact in fp32; a sum may lose 2^-16 of the sum of the sizes, and the bf16 result is rounded to 8 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(M, K, N, bias=False, seed=0):
    from autodist_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + M * 1009 + K * 31 + N)
    x, w = torch.randn(M, K, generator=g, device="cuda"), torch.randn(N, K, generator=g, device="cuda")
    x *= torch.rand(M, 1, generator=g, device="cuda") * 4
    return F.quantize_rows(x) + F.quantize_rows(w) + (torch.randn(N, generator=g, device="cuda") if bias else None,)


def _check(args, y=None):
    from autodist_b200.ops import functional as F
    codes, scales, weight, weight_scales, bias = args
    y = F.linear_8bit(*args) if y is None else y
    assert y.dtype == torch.bfloat16 and y.shape == codes.shape[:-1] + weight.shape[:1]
    a, b = codes.double() * scales.double()[..., None], weight.double() * weight_scales.double()[:, None]
    want = a @ b.t()
    sizes = a.abs() @ b.abs().t()
    if bias is not None:
        want, sizes = want + bias.double(), sizes + bias.double().abs()
    off = (y.double() - want).abs() - 2.0 ** -8 * want.abs() - 2.0 ** -16 * sizes - 1e-37
    assert not torch.isnan(off).any() and (not off.numel() or float(off.max()) <= 0), float(off.max())


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 127, 128, 129, 200, 255, 257, 300, 513])
@pytest.mark.parametrize("K,N", [(64, 64), (128, 96), (256, 1000), (1000, 130), (1001, 257), (2048, 512), (33, 17)])
def test_shapes(M, K, N):
    _check(_inputs(M, K, N, bias=M % 2 == 0))


@pytest.mark.parametrize("K", [1, 2, 15, 16, 17, 31, 32, 127, 128, 129, 255, 257, 4095, 4097])
@pytest.mark.parametrize("M,N", [(1, 1), (5, 40), (130, 300)])
def test_contractions(K, M, N):
    _check(_inputs(M, K, N))


@pytest.mark.parametrize("N", [1, 2, 7, 8, 15, 31, 63, 127, 129, 256, 1025])
@pytest.mark.parametrize("M", [1, 40, 260])
def test_outputs(M, N):
    _check(_inputs(M, 272, N, bias=True))


@pytest.mark.parametrize("M,K,N", [(1024, 1024, 2048), (4096, 512, 1536), (2000, 1500, 4000), (777, 4096, 8200), (16, 16384, 640), (2, 64, 30522), (8, 2048, 8192),
                                   (3000, 2100, 260), (5000, 96, 5000)])
def test_large(M, K, N):
    args = _inputs(M, K, N, bias=True)
    _check(args)
    from autodist_b200.ops import functional as F
    assert torch.equal(F.linear_8bit(*args), F.linear_8bit(*args))


@pytest.mark.parametrize("bn", [16, 32, 64, 128, 512])
@pytest.mark.parametrize("M,K,N", [(1, 1100, 130), (37, 2304, 264), (150, 1024, 1003), (300, 640, 520)])
def test_every_tile_and_share(bn, M, K, N):
    from autodist_b200 import ops
    from autodist_b200.ops import functional as F
    E, args = ops.ext(required=True), _inputs(M, K, N, bias=True)
    err = F._error_flag(args[0].device)
    for split in (1, 2, 3, 4, 5, 6, 7, 8) if bn != 512 else (1,):
        if split <= (K + 127) // 128:
            _check(args, E.gemm_8bit(*args, err, bn, split))
        else:
            with pytest.raises(RuntimeError, match="invalid"):
                E.gemm_8bit(*args, err, bn, split)
    F.check_errors()


def test_codes_of_every_value():
    """All 256 codes: NaN rows give NaN, everything else its value."""
    from autodist_b200.ops import functional as F
    codes = torch.arange(256, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    w = torch.zeros(32, 16, device="cuda").to(torch.float8_e4m3fn)
    w[:, 0] = torch.ones((), device="cuda").to(torch.float8_e4m3fn)
    x = torch.zeros(256, 16, device="cuda").to(torch.float8_e4m3fn)
    x[:, 0] = codes
    y = F.linear_8bit(x, torch.ones(256, device="cuda"), w, torch.ones(32, device="cuda"))
    want = codes.float()[:, None].expand(256, 32)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.float().nan_to_num(), want.nan_to_num())


def test_scales_that_are_not_finite_or_zero():
    from autodist_b200.ops import functional as F
    codes, scales, weight, weight_scales, _ = _inputs(20, 96, 48)
    clean = F.linear_8bit(codes, scales, weight, weight_scales)
    scales[3], scales[5] = float("nan"), 0.0
    y = F.linear_8bit(codes, scales, weight, weight_scales)
    assert y[3].isnan().all() and (y[5] == 0).all()
    others = [i for i in range(20) if i not in (3, 5)]
    assert torch.equal(y[others], clean[others])
    # large scales on one side, small ones on the other: their product is what counts
    y = F.linear_8bit(codes[others], scales[others] * 1e30, weight, weight_scales * 1e-30)
    assert torch.allclose(y.float(), clean[others].float(), rtol=2.0 ** -7)


def test_rows_that_the_kernel_cannot_read_in_place():
    from autodist_b200.ops import functional as F
    codes, scales, weight, weight_scales, bias = _inputs(50, 100, 70, bias=True)
    want = F.linear_8bit(codes, scales, weight, weight_scales, bias)
    wide = torch.zeros(50, 321, device="cuda").to(torch.float8_e4m3fn)
    wide[:, 3:103] = codes
    views = [codes.contiguous(), wide[:, 3:103], codes.t().contiguous().t(), torch.cat([codes] * 2, 0)[:50]]
    for v in views:
        assert torch.equal(F.linear_8bit(v, scales, weight, weight_scales, bias), want)
        assert torch.equal(F.linear_8bit(codes.unflatten(0, (5, 10)), scales.view(5, 10), weight, weight_scales, bias).view_as(want), want)
    assert torch.equal(F.linear_8bit(codes, scales, weight.contiguous(), weight_scales, bias), want)
    assert torch.equal(F.linear_8bit(codes[::2], scales[::2], weight, weight_scales, bias), want[::2])
    assert torch.equal(F.linear_8bit(codes[7:8], scales[7:8], weight, weight_scales, bias), want[7:8])
    one = F.linear_8bit(codes[:1].expand(9, 100), scales[:1].expand(9), weight, weight_scales, bias)
    assert torch.equal(one, want[:1].expand(9, 70))


def test_no_rows_or_outputs():
    from autodist_b200.ops import functional as F
    codes, scales, weight, weight_scales, bias = _inputs(5, 64, 32, bias=True)
    assert F.linear_8bit(codes[:0], scales[:0], weight, weight_scales, bias).shape == (0, 32)
    assert F.linear_8bit(codes, scales, weight[:0], weight_scales[:0]).shape == (5, 0)


def test_behind_the_norm():
    from autodist_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(2)
    x, r = (torch.randn(2, 19, 520, generator=g, device="cuda").bfloat16() for _ in range(2))
    w, weight = torch.rand(520, generator=g, device="cuda") + 0.5, torch.randn(264, 520, generator=g, device="cuda") / 23
    codes, scales, s = F.rms_norm_8bit(x, w, r)
    y = F.linear_8bit(codes, scales, *F.quantize_rows(weight))
    assert y.shape == (2, 19, 264)
    full = F.rms_norm(x, w, r)[0].float() @ weight.t()
    # each side is off by 2^-5 of an element at most in the mean square: sqrt(2) of that between them
    assert float((y.float() - full).norm() / full.norm()) < 2.0 ** -4


def test_on_another_stream():
    from autodist_b200.ops import functional as F
    for shape in ((300, 512, 512), (8, 512, 2048), (2048, 1024, 2048)):
        args = _inputs(*shape)
        want = F.linear_8bit(*args)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = F.linear_8bit(*args)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
    F.check_errors()


def test_offsets_past_31_bits():
    """More than 2^31 outputs, and more than 2^31 bytes of weights."""
    from autodist_b200.ops import functional as F
    M, K, N = 70000, 64, 32768
    args = _inputs(M, K, N)
    y = F.linear_8bit(*args)
    few = F.linear_8bit(args[0][-5:], args[1][-5:], *args[2:])
    assert torch.allclose(y[-5:].float(), few.float(), rtol=2.0 ** -7, atol=1e-3)
    del y, few
    wide = torch.zeros(2 ** 20 + 8, 2048, dtype=torch.float8_e4m3fn, device="cuda")
    weight = torch.randn(8, 2048, device="cuda")
    wide[-8:], scale = F.quantize_rows(weight)
    scales = torch.ones(2 ** 20 + 8, device="cuda")
    scales[-8:] = scale
    x, sx = F.quantize_rows(torch.randn(3, 2048, device="cuda"))
    y = F.linear_8bit(x, sx, wide, scales)
    assert not y[:, :-8].any()
    _check((x, sx, wide[-8:], scale, None), y[:, -8:])


def test_refusals():
    from autodist_b200.ops import functional as F
    codes, scales, weight, weight_scales, bias = _inputs(5, 64, 32, bias=True)
    for bad in ((codes.float(), scales, weight, weight_scales), (codes, scales, weight.view(torch.uint8), weight_scales)):
        with pytest.raises(TypeError, match="float8_e4m3fn"):
            F.linear_8bit(*bad)
    with pytest.raises(ValueError, match="do not match"):
        F.linear_8bit(codes[:, :63], scales, weight, weight_scales)
    with pytest.raises(ValueError, match="do not match"):
        F.linear_8bit(codes[:, :0], scales, weight[:, :0], weight_scales)
    for bad in ((codes, scales[:4], weight, weight_scales), (codes, scales, weight, weight_scales.double()), (codes, scales[:, None], weight, weight_scales)):
        with pytest.raises(ValueError, match="scale for each row"):
            F.linear_8bit(*bad)
    from autodist_b200 import ops
    for bn, split in ((17, 1), (128, 9), (128, 2)):
        with pytest.raises(RuntimeError, match="invalid"):
            ops.ext(required=True).gemm_8bit(codes, scales, weight, weight_scales, None, F._error_flag(codes.device), bn, split)
    with pytest.raises(ValueError, match="bias"):
        F.linear_8bit(codes, scales, weight, weight_scales, bias.bfloat16())
    with pytest.raises(RuntimeError, match="no gradient"):
        F.linear_8bit(codes, scales.clone().requires_grad_(True), weight, weight_scales)
    for bad in ((codes, scales.cpu(), weight, weight_scales), (codes, scales, weight.cpu(), weight_scales), (codes, scales, weight, weight_scales, bias.cpu())):
        with pytest.raises(RuntimeError, match="GPU"):
            F.linear_8bit(*bad)
