"""The gated recurrence against a walk through time in 64 bits.

A step adds an error of a few fp32 roundings of f h and u x to what it carries on, sigmoids included (their exponentials lose about a
rounding for each unit of the argument): UNIT covers 24 roundings. ``_Walk`` carries the sum of those sizes along, so that the bound is the
recurrence's own; bf16 results add 2^-8 of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = 24 * 2.0 ** -24
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -22}


def _inputs(batch, steps, channels, dtype, gate=False, state=True, resets=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + batch * 10007 + steps * 101 + channels)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    keep = torch.empty(channels, device="cuda").uniform_(-1, 6, generator=g)
    s = {"x": normal(batch, steps, channels).to(dtype), "forget": (normal(batch, steps, channels) + keep).to(dtype),
         "input_gate": normal(batch, steps, channels).to(dtype) if gate else None, "state": normal(batch, channels) if state else None, "reset": None}
    if resets is not None:
        s["reset"] = torch.rand(batch, steps, generator=g, device="cuda") < resets
    s["dy"], s["dlast"] = normal(batch, steps, channels).to(dtype), normal(batch, channels)
    return s


class _Walk:
    """Outputs, gradients and what they may be off, in 64 bits."""

    def __init__(self, s, bias=0.0):
        x, a = s["x"].double(), s["forget"].double() + bias
        B, T, C = x.shape
        f, nf = torch.sigmoid(a), torch.sigmoid(-a)
        u, nu = (nf, f) if s["input_gate"] is None else (torch.sigmoid(s["input_gate"].double()), torch.sigmoid(-s["input_gate"].double()))
        cut = torch.zeros(B, T, dtype=torch.bool, device=x.device) if s["reset"] is None else s["reset"]
        h = torch.zeros(B, C, dtype=torch.float64, device=x.device) if s["state"] is None else s["state"].double()
        most, off = h.abs(), torch.zeros_like(h)             # the largest that h can be, and what may be wrong with it
        self.y, self.off, before, most_before, off_before = [], [], [], [], []
        for t in range(T):
            held = torch.where(cut[:, t, None], 0.0, f[:, t])
            before.append(torch.where(cut[:, t, None], 0.0, h))
            most_before.append(torch.where(cut[:, t, None], 0.0, most))
            off_before.append(torch.where(cut[:, t, None], 0.0, off))
            v = u[:, t] * x[:, t]
            off = held * off + UNIT * (held * most + v.abs())
            most = held * most + v.abs()
            h = held * h + v
            self.y.append(h)
            self.off.append(off)
        self.last, self.last_off = h, off
        self.y = torch.stack(self.y, 1) if T else x
        self.off = torch.stack(self.off, 1) if T else x
        dh, dmost, doff = s["dlast"].double(), s["dlast"].double().abs(), torch.zeros(B, C, dtype=torch.float64, device=x.device)
        g = {k: torch.zeros_like(x) for k in ("x", "forget", "input_gate")}
        o = {k: torch.zeros_like(x) for k in ("x", "forget", "input_gate")}
        for t in range(T - 1, -1, -1):
            dy = s["dy"][:, t].double()
            doff = doff + UNIT * (dmost + dy.abs())
            dmost, dh = dmost + dy.abs(), dh + dy
            hb, mb, ob = before[t], most_before[t], off_before[t]
            xt = x[:, t]
            slope = f[:, t] * nf[:, t]
            g["x"][:, t], o["x"][:, t] = dh * u[:, t], doff * u[:, t] + UNIT * dmost * u[:, t]
            coupled = s["input_gate"] is None
            g["forget"][:, t] = dh * (hb - xt if coupled else hb) * slope
            sizes = mb + (xt.abs() if coupled else 0)
            o["forget"][:, t] = (doff * sizes + dmost * ob + UNIT * dmost * sizes) * slope
            if not coupled:
                g["input_gate"][:, t] = dh * xt * u[:, t] * nu[:, t]
                o["input_gate"][:, t] = (doff + UNIT * dmost) * xt.abs() * u[:, t] * nu[:, t]
            held = torch.where(cut[:, t, None], 0.0, f[:, t])
            dh, dmost, doff = dh * held, dmost * held, doff * held + UNIT * dmost * held
        self.grads, self.offs, self.dstate, self.dstate_off = g, o, dh, doff


def _near(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound - 1e-36             # (results below the normal range)
    assert not torch.isnan(off).any() and (not off.numel() or float(off.max()) <= 0), float(off.max())


def _alike(a, b):
    """Two ways to split the same recurrence: each may be off by its bound."""
    _near(a, b.double(), 2 * ROUND[a.dtype] * b.double().abs() + 1e-4 * float(b.double().abs().max()))


def _check(s, bias=0.0):
    from autodist_b200.ops import functional as F
    dtype, walk = s["x"].dtype, _Walk(s, bias)
    args = [s["x"], s["forget"], s["input_gate"], s["state"], s["reset"], bias]
    with torch.no_grad():
        y, last = F.gated_recurrence(*args)
    assert y.dtype == dtype and last.dtype == torch.float32
    _near(y, walk.y, walk.off + ROUND[dtype] * (walk.y.abs() + walk.off))
    _near(last, walk.last, walk.last_off)
    leaves = {k: s[k].detach().requires_grad_(True) for k in ("x", "forget", "input_gate", "state") if s[k] is not None}
    y2, last2 = F.gated_recurrence(*(leaves.get(k, s[k]) for k in ("x", "forget", "input_gate", "state", "reset")), bias)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    grads = dict(zip(leaves, torch.autograd.grad((y2, last2), list(leaves.values()), (s["dy"], s["dlast"]))))
    for k in ("x", "forget", "input_gate"):
        if k in grads:
            assert grads[k].dtype == dtype
            _near(grads[k], walk.grads[k], 2 * walk.offs[k] + ROUND[dtype] * (walk.grads[k].abs() + walk.offs[k]))
    if "state" in grads:
        _near(grads["state"], walk.dstate, walk.dstate_off)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 33, 64, 65, 127, 128, 129, 255, 257, 300, 1025])
def test_lengths(dtype, gate, steps):
    _check(_inputs(2, steps, 72, dtype, gate, state=steps % 2 == 1, resets=0.03 if steps % 3 == 0 else None))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("batch,channels", [(1, 1), (3, 2), (1, 31), (2, 33), (1, 64), (5, 66), (1, 127), (2, 130), (1, 515), (40, 96), (1, 1024)])
def test_channels(dtype, gate, batch, channels):
    _check(_inputs(batch, 141, channels, dtype, gate, resets=0.02))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,steps,channels", [(1, 9000, 64), (1, 5001, 130), (2, 4097, 33), (1, 33000, 8), (160, 40, 256), (300, 5, 130), (1, 2500, 2048)])
def test_shapes_that_are_split_in_their_own_way(dtype, batch, steps, channels):
    _check(_inputs(batch, steps, channels, dtype, gate=batch % 2 == 0, resets=0.001))


@pytest.mark.parametrize("resets", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("steps", [1, 4, 5, 200, 1500])
def test_resets(resets, steps):
    s = _inputs(2, steps, 70, torch.float32, resets=resets)
    _check(s)
    if resets == 1.0:
        from autodist_b200.ops import functional as F
        y, _ = F.gated_recurrence(s["x"], s["forget"], reset=s["reset"], state=torch.full_like(s["state"], float("inf")))
        assert y.isfinite().all()                           # nothing of the state is left, infinite as it may be


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("steps", [1, 40, 700])
def test_gates_at_their_limits(dtype, steps):
    """Gates of infinities and of the type's lowest value: shut is zero, open is one."""
    from autodist_b200.ops import functional as F
    s = _inputs(2, steps, 66, dtype, gate=True)
    low = torch.finfo(dtype).min
    for shut in (low, float("-inf")):
        y, last = F.gated_recurrence(s["x"], torch.full_like(s["forget"], shut), s["input_gate"], s["state"])
        want = (torch.sigmoid(s["input_gate"].double()) * s["x"].double())
        _near(y, want, (ROUND[dtype] + UNIT) * want.abs())
        y, last = F.gated_recurrence(s["x"], torch.full_like(s["forget"], -shut), torch.full_like(s["x"], shut), s["state"])
        assert torch.equal(last, s["state"]) and torch.equal(y, s["state"][:, None].expand_as(y).to(dtype))
        y, last = F.gated_recurrence(s["x"], torch.full_like(s["forget"], -shut), None, s["state"])
        assert torch.equal(last, s["state"])
    leaves = [t.requires_grad_(True) for t in (s["x"], torch.full_like(s["forget"], low), torch.full_like(s["forget"], float("inf")))]
    y, last = F.gated_recurrence(*leaves, s["state"])
    for g in torch.autograd.grad((y, last), leaves, (s["dy"], s["dlast"])):
        assert g.isfinite().all()


def test_what_is_not_finite_stays_in_its_channel_and_behind_a_reset():
    from autodist_b200.ops import functional as F
    s = _inputs(2, 900, 70, torch.float32)
    reset = torch.zeros(2, 900, dtype=torch.bool, device="cuda")
    reset[0, 400] = True
    y, last = F.gated_recurrence(s["x"], s["forget"], None, s["state"], reset)
    x = s["x"].clone()
    x[0, 100, 3], x[0, 120, 5] = float("nan"), float("inf")
    bad, bad_last = F.gated_recurrence(x, s["forget"], None, s["state"], reset)
    others = [c for c in range(70) if c not in (3, 5)]
    assert torch.equal(bad[:, :, others], y[:, :, others]) and torch.equal(bad[1], y[1]) and torch.equal(bad[0, 400:], y[0, 400:]) and torch.equal(bad_last, last)
    assert bad[0, 100:400, 3].isnan().all() and torch.equal(bad[0, :100, 3], y[0, :100, 3])


def test_a_sequence_in_pieces_is_the_sequence():
    """Prompt first, then token by token with the state passed on."""
    from autodist_b200.ops import functional as F
    s = _inputs(3, 150, 96, torch.float32, gate=True)
    walk = _Walk(s)
    state, outs = s["state"], []
    for a, b in [(0, 130)] + [(t, t + 1) for t in range(130, 140)] + [(140, 150)]:
        y, state = F.gated_recurrence(s["x"][:, a:b], s["forget"][:, a:b], s["input_gate"][:, a:b], state)
        outs.append(y)
    _near(torch.cat(outs, 1), walk.y, 2 * walk.off + ROUND[torch.float32] * walk.y.abs())
    _near(state, walk.last, 2 * walk.last_off)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("channels", [64, 33])
def test_strided_views(dtype, channels):
    from autodist_b200.ops import functional as F
    s = _inputs(3, 210, 3 * channels + 1, dtype, resets=0.01)
    whole = s["x"]
    for off in (0, 1):
        x, f, i = (whole[..., off + k * channels:off + (k + 1) * channels] for k in range(3))
        views = [(x, f, i), tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, f, i)), (x[:, :1].expand_as(x), f, i),
                 tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x, f, i))]
        for v in views:
            dense = [t.contiguous() for t in v]
            reset = s["reset"].t().contiguous().t()
            args = [t.detach().requires_grad_(True) for t in v], [t.detach().clone().requires_grad_(True) for t in dense]
            got, want = (F.gated_recurrence(*a, None, r) for a, r in zip(args, (reset, s["reset"])))
            for a, b in zip(got, want):
                _alike(a, b)
            dy = s["dy"][..., :channels]
            for a, b in zip(torch.autograd.grad(got[0], args[0], dy), torch.autograd.grad(want[0], args[1], dy.contiguous())):
                _alike(a, b)


def test_a_sum_that_only_reads_the_last_state_or_the_outputs():
    from autodist_b200.ops import functional as F
    s = _inputs(2, 77, 40, torch.float32)
    x = s["x"].requires_grad_(True)
    y, last = F.gated_recurrence(x, s["forget"], None, s["state"])
    a, = torch.autograd.grad(last, x, s["dlast"], retain_graph=True)
    b, = torch.autograd.grad(y, x, s["dy"], retain_graph=True)
    both, = torch.autograd.grad((y, last), x, (s["dy"], s["dlast"]), retain_graph=True)
    _near(both, a.double() + b.double(), 1e-5 * (a.double().abs() + b.double().abs()) + 1e-6)
    ones, = torch.autograd.grad(y.sum(), x)
    assert ones.isfinite().all()


def test_empty():
    from autodist_b200.ops import functional as F
    state = torch.randn(2, 8, device="cuda", requires_grad=True)
    x = torch.zeros(2, 0, 8, device="cuda", requires_grad=True)
    y, last = F.gated_recurrence(x, x, state=state)
    assert y.shape == (2, 0, 8) and torch.equal(last, state)
    assert torch.equal(torch.autograd.grad(last, state, torch.ones_like(last))[0], torch.ones_like(last))
    y, last = F.gated_recurrence(torch.zeros(0, 5, 8, device="cuda"), torch.zeros(0, 5, 8, device="cuda"))
    assert y.shape == (0, 5, 8) and last.shape == (0, 8)
    y, last = F.gated_recurrence(torch.zeros(2, 0, 8, device="cuda"), torch.zeros(2, 0, 8, device="cuda"))
    assert (last == 0).all()


def test_against_differences_and_second_derivatives():
    from autodist_b200.ops import functional as F
    s = _inputs(2, 19, 5, torch.float32, gate=True, resets=0.1)
    names = ("x", "forget", "input_gate", "state")
    leaves = [s[k].requires_grad_(True) for k in names]
    grads = torch.autograd.grad(F.gated_recurrence(*leaves, s["reset"], 0.5), leaves, (s["dy"], s["dlast"]))
    g = torch.Generator(device="cuda").manual_seed(3)
    steps = [torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64) for t in leaves]

    def value(h):
        moved = {k: t.detach().double() + h * d for k, t, d in zip(names, leaves, steps)}
        walk = _Walk(dict(moved, reset=s["reset"], dy=s["dy"], dlast=s["dlast"]), 0.5)
        return float((walk.y * s["dy"].double()).sum() + (walk.last * s["dlast"].double()).sum())
    slope = (value(1e-5) - value(-1e-5)) / 2e-5
    sizes = sum(float((a.double() * d).abs().sum()) for a, d in zip(grads, steps))
    assert abs(sum(float((a.double() * d).sum()) for a, d in zip(grads, steps)) - slope) <= 1e-5 * sizes

    def twice(leaves, reset):
        first = torch.autograd.grad(F.gated_recurrence(*leaves, reset)[0].square().sum(), leaves, create_graph=True)
        return torch.autograd.grad(sum((f * f).sum() for f in first), leaves)
    there = twice([t.detach().clone().requires_grad_(True) for t in leaves], s["reset"])
    here = twice([t.detach().cpu().requires_grad_(True) for t in leaves], s["reset"].cpu())
    for a, b in zip(there, here):
        assert torch.allclose(a.cpu(), b, rtol=1e-3, atol=1e-3 * float(b.abs().max()))


@pytest.mark.parametrize("batch,steps,channels", [(4, 70, 64), (1, 6000, 256)])
def test_on_another_stream_and_twice(batch, steps, channels):
    from autodist_b200.ops import functional as F
    s = _inputs(batch, steps, channels, torch.bfloat16)
    leaves = [s["x"].requires_grad_(True), s["forget"].requires_grad_(True)]

    def once():
        out = F.gated_recurrence(*leaves, None, s["state"])
        return out + torch.autograd.grad(out, leaves, (s["dy"], s["dlast"]))
    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_31_bits():
    from autodist_b200.ops import functional as F
    batch, steps, channels = 3, 11000, 2 ** 16 + 2
    x = torch.randn(1, 1, channels, device="cuda").bfloat16().expand(batch, steps, channels)
    forget = torch.zeros(1, 1, channels, dtype=torch.bfloat16, device="cuda").expand(batch, steps, channels)
    y, last = F.gated_recurrence(x, forget)
    small, small_last = F.gated_recurrence(x[:1, :, -64:], forget[:1, :, -64:])
    _alike(y[2, :, -64:], small[0])
    _alike(last[2, -64:], small_last[0])


def test_refusals():
    from autodist_b200 import ops
    from autodist_b200.ops import functional as F
    x, state, reset = torch.ones(2, 4, 8, device="cuda"), torch.ones(2, 8, device="cuda"), torch.zeros(2, 4, dtype=torch.bool, device="cuda")
    with pytest.raises(TypeError, match="bf16 or fp32"):
        F.gated_recurrence(x.half(), x.half())
    with pytest.raises(ValueError, match="batch, steps, channels"):
        F.gated_recurrence(x[0], x[0])
    for args in ((x, x[:, :3]), (x, x.bfloat16()), (x, x, x[:1])):
        with pytest.raises(ValueError, match="gate must have"):
            F.gated_recurrence(*args)
    for bad in (state.bfloat16(), state[:1], state[:, :7]):
        with pytest.raises(ValueError, match="fp32 state"):
            F.gated_recurrence(x, x, state=bad)
    for bad in (reset.int(), reset[:, :3]):
        with pytest.raises(ValueError, match="bool reset"):
            F.gated_recurrence(x, x, reset=bad)
    for args in ((x, x.cpu()), (x, x, None, state.cpu()), (x, x, None, None, reset.cpu())):
        with pytest.raises(RuntimeError, match="GPU"):
            F.gated_recurrence(*args)
    for bad in (float("inf"), float("nan")):
        with pytest.raises(ValueError, match="finite forget_bias"):
            F.gated_recurrence(x, x, forget_bias=bad)
    E = ops.ext(required=True)
    with pytest.raises(RuntimeError, match="GPU"):
        E.gated_scan_fwd(x.cpu(), x, None, None, None, 0.0, False)
    with pytest.raises(RuntimeError, match="states needed"):
        E.gated_scan_bwd(x, None, x, x, None, None, None, torch.zeros(3, device="cuda"), 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("batch,steps,channels", [(2, 1, 8), (3, 37, 33), (1, 3001, 64)])
def test_training_calls_leave_their_inputs_alone(batch, steps, channels, gate, dtype):
    from autodist_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(steps)
    x, forget, i, dy = (torch.randn(batch, steps, channels, generator=g, device="cuda").to(dtype) for _ in range(4))
    state, dlast = (torch.randn(batch, channels, generator=g, device="cuda") for _ in range(2))
    inputs = [x, forget, state, dy, dlast] + ([i] if gate else [])
    before = [t.clone() for t in inputs]
    leaves = [t.requires_grad_(True) for t in ([x, forget, i, state] if gate else [x, forget, state])]
    results = []
    for _ in range(3):
        out = F.gated_recurrence(x, forget, i if gate else None, state=state)
        results.append(list(out) + list(torch.autograd.grad(out, leaves, (dy, dlast))))
    assert all(torch.equal(a, b.detach()) for a, b in zip(before, inputs))
    assert all(torch.equal(a, b) for later in results[1:] for a, b in zip(results[0], later))
