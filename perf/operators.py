"""What the operators of a gated recurrent language model are timed on: its norm (trained, and with an output in 8 bits), its recurrence
over time, the product of 8-bit rows that reads the norm's output, and the optimizer step over its list of parameters.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` builds what a user's program holds before
the call, ``run`` is one call, ``work`` the bytes and operations that one call cannot do without and ``exact`` its outputs in 64 bits.
``own`` chooses between the framework's operators and their plain forms: elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
E4M3_MAX = 448.0
BLOCK = 256                     # elements of a tensor that share a scale of the optimizer's 8-bit states
TINIEST = 2.0 ** -100           # moments below are held as zeros in 8 bits
EPS = 1e-6                      # of the norm
ADAMW = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}
OPT_SEED, OPT_STEP = 11, 40     # the optimizer's seed, and how many steps it has behind it

# the largest listed cases, which bound what draw() asks for
MOST_NORM, MOST_SCAN, MOST_MACS, MOST_PARAMS = 16384 * 4096, 65536 * 1024, 8192 * 4096 * 4096, 120_000_000


def _case(name, op, **values):
    return dict(values, op=op, name=name) if name else dict(values, op=op)


def _norm(name, form, rows, width, dtype="bf16", residual=True):
    return _case(name, "norm", form=form, rows=rows, width=width, dtype=dtype, residual=residual)


def _scan(name, form, batch, steps, channels, dtype="bf16", input_gate=False, resets=False):
    return _case(name, "scan", form=form, batch=batch, steps=steps, channels=channels, dtype=dtype, input_gate=input_gate, resets=resets)


def _linear(name, rows, inputs, outputs, bias=False):
    return _case(name, "linear", rows=rows, inputs=inputs, outputs=outputs, bias=bias)


def _adamw(name, bits, hidden, layers, vocab, dtype="fp32", align=256):
    return _case(name, "adamw", bits=bits, hidden=hidden, layers=layers, vocab=vocab, dtype=dtype, align=align)


def listed():
    return [
        # one decoding step of 8 sequences: the residual stream is added and normed into the 8-bit rows that the next product reads
        _norm("norm_8bit_step", "8bit", 8, 2048),
        # the same over a batch of long prompts
        _norm("norm_8bit_prompt", "8bit", 16384, 4096),
        # a training step's norm at the width and tokens of BERT-large's batch, forward and backward
        _norm("norm_train", "train", 4096, 1024),
        # full precision on an odd width and an odd number of rows, without a residual, forward and backward
        _norm("norm_train_fp32_odd", "train", 12289, 1001, "fp32", residual=False),
        # one token of each of 128 sequences: the serving form
        _scan("scan_token", "forward", 128, 1, 2048, input_gate=True),
        # the LM1B training batch, 128 x 20 tokens with 2048 units, both gates
        _scan("scan_train_lm1b", "train", 128, 20, 2048, input_gate=True),
        # one long document: parallelism has to come from time
        _scan("scan_train_long", "train", 1, 65536, 1024),
        # packed prompts in full precision: state forgotten where a document begins, odd numbers of steps and channels
        _scan("scan_packed_fp32_odd", "forward", 3, 4099, 515, "fp32", resets=True),
        # one decoding step of 8 sequences through a projection: the weight's bytes are what counts
        _linear("linear_step", 8, 2048, 8192),
        # a batch of long prompts through a projection
        _linear("linear_prompt", 8192, 4096, 4096, bias=True),
        # the optimizer step of a model of 18 blocks, moments in 8 bits
        _adamw("adamw_8bit", 8, 1024, 18, 30522),
        # a small model's many small tensors of odd sizes, packed without alignment, moments in 32 bits
        _adamw("adamw_small_odd", 32, 61, 12, 997, align=1),
    ]


def _spread(rng, low, high):
    """A whole number between ``low`` and ``high``, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _sized(rng, low, high):
    """Half of the sizes as they fall, half of them multiples of 8."""
    n = _spread(rng, low, high)
    n = n if rng.random() < 0.5 else max(low, min(high, -(-n // 8) * 8))
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(("norm", "scan", "linear", "adamw"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if op == "norm":
        width = _sized(rng, 16, 8192)
        rows = _spread(rng, 1, max(1, min(32768, MOST_NORM // (2 * width))))
        form = rng.choice(("8bit", "train"))
        return _norm(None, form, rows, width, dtype, rng.random() < 0.7)
    if op == "scan":
        channels = _sized(rng, 32, 4096)
        steps = _spread(rng, 1, min(65536, MOST_SCAN // (2 * channels)))
        batch = _spread(rng, 1, max(1, min(128, MOST_SCAN // (2 * channels * steps))))
        return _scan(None, rng.choice(("forward", "train")), batch, steps, channels, dtype, rng.random() < 0.5, rng.random() < 0.4)
    if op == "linear":
        inputs, outputs = _sized(rng, 64, 4096), _sized(rng, 64, 8192)
        return _linear(None, _spread(rng, 1, min(8192, MOST_MACS // (inputs * outputs))), inputs, outputs, rng.random() < 0.5)
    hidden, layers = _spread(rng, 24, 1024), rng.randint(2, 16)
    vocab = _spread(rng, 100, 30000)
    while sum(_sizes(hidden, layers, vocab)) > MOST_PARAMS:
        layers, vocab = max(1, layers // 2), vocab // 2
    align = rng.choice((1, 8, 256)) if hidden <= 256 else 256
    return _adamw(None, rng.choice((8, 8, 32)), hidden, layers, vocab, dtype, align)


def _sizes(hidden, layers, vocab):
    """Elements of each parameter: embedding, then per block the norm, the projection into twice as many units and their gates, and back."""
    block = [hidden, 2 * (2 * hidden) * hidden, 4 * hidden, hidden * 2 * hidden]
    return [vocab * hidden] + block * layers + [hidden]


# ---------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return torch.randn(*shape, generator=g, device=DEVICE).mul_(scale).add_(shift).to(dtype)


def _codes(x):
    """Rows of ``x`` as e4m3 values and a scale each; rows start on 16-byte boundaries, as the framework lays them out."""
    rows, width = x.shape
    scale = x.abs().amax(1) / E4M3_MAX
    out = torch.zeros(rows, -(-width // 16) * 16, dtype=torch.float8_e4m3fn, device=x.device)[:, :width]
    return out.copy_((x / scale.clamp_min(1e-30)[:, None]).to(torch.float8_e4m3fn)), scale


def prepare(case, seed):
    g = _generator(seed)
    return {"norm": _prepare_norm, "scan": _prepare_scan, "linear": _prepare_linear, "adamw": _prepare_adamw}[case["op"]](case, g)


def _prepare_norm(case, g):
    rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
    train = case["form"] == "train"
    # a residual stream: a few channels are much larger than the others
    outliers = 1.0 + 20.0 * (torch.rand(width, generator=g, device=DEVICE) < 0.01)
    s = {"case": case, "x": (_normal(g, rows, width) * outliers).to(dtype), "weight": _normal(g, width, scale=0.1, shift=1.0), "residual": None}
    if case["residual"]:
        s["residual"] = (_normal(g, rows, width, scale=2.0) * outliers).to(dtype)
    if train:
        s["dy"] = _normal(g, rows, width, dtype=dtype)
        s["ds"] = _normal(g, rows, width, dtype=dtype) if case["residual"] else None
        for k in ("x", "weight", "residual"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def _prepare_scan(case, g):
    batch, steps, channels, dtype = case["batch"], case["steps"], case["channels"], DTYPES[case["dtype"]]
    shape = (batch, steps, channels)
    # forget gates of a trained model: most channels keep their state for tens to thousands of steps
    keep = torch.empty(channels, device=DEVICE).uniform_(0.0, 7.0, generator=g)
    s = {"case": case, "x": _normal(g, *shape, dtype=dtype), "forget": (_normal(g, *shape) + keep).to(dtype), "input": None, "reset": None,
         "state": _normal(g, batch, channels)}
    if case["input_gate"]:
        s["input"] = _normal(g, *shape, dtype=dtype)
    if case["resets"]:
        s["reset"] = torch.rand(batch, steps, generator=g, device=DEVICE) < 0.003
    if case["form"] == "train":
        s["dy"], s["dlast"] = _normal(g, *shape, dtype=dtype), _normal(g, batch, channels)
        for k in ("x", "forget", "input", "state"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def _prepare_linear(case, g):
    x, w = _normal(g, case["rows"], case["inputs"]), _normal(g, case["outputs"], case["inputs"], scale=case["inputs"] ** -0.5)
    s = {"case": case, "bias": _normal(g, case["outputs"]) if case["bias"] else None}
    s["codes"], s["scales"] = _codes(x)
    s["weight_codes"], s["weight_scales"] = _codes(w)
    return s


def _prepare_adamw(case, g):
    sizes, dtype, bits = _sizes(case["hidden"], case["layers"], case["vocab"]), DTYPES[case["dtype"]], case["bits"]
    starts, total = _starts(sizes, case["align"])
    places, padded = _starts(sizes, BLOCK)          # where the tensors' states lie
    values, grads = _normal(g, total, dtype=dtype, scale=0.02), _normal(g, total, dtype=dtype, scale=1e-3)
    filled = torch.zeros(padded, dtype=torch.bool, device=DEVICE)
    for o, n in zip(places, sizes):
        filled[o:o + n] = True
    if case["align"] == BLOCK:                      # nothing lies between the tensors
        values.mul_(filled)
        grads.mul_(filled)
    params = [torch.nn.Parameter(values[o:o + n]) for o, n in zip(starts, sizes)]
    for p, o, n in zip(params, starts, sizes):
        p.grad = grads[o:o + n]
    m, r = _normal(g, padded, scale=1e-4) * filled, _normal(g, padded, scale=1e-3).abs_().add_(1e-6) * filled
    s = {"case": case, "values": values, "step": OPT_STEP, "grads": grads, "params": params, "index": None, "filled": None}
    if case["align"] != BLOCK:
        # tensors packed closer than their states: where each state's parameter lies
        s["index"] = torch.cat([torch.arange(o, o + -(-n // BLOCK) * BLOCK, device=DEVICE) for o, n in zip(starts, sizes)]).clamp_(max=total - 1)
        s["filled"] = filled
    if bits == 8:
        s["exp_avg"], s["exp_avg_scale"] = _nearest(m)
        s["exp_avg_sq"], s["exp_avg_sq_scale"] = _nearest(r)
    else:
        s["exp_avg"], s["exp_avg_sq"] = m, r * r
    if own:
        from autodist_b200.optim import ListAdamW
        s["optimizer"] = ListAdamW(params, state_bits=bits, seed=OPT_SEED, **ADAMW)
        s["optimizer"].load_buffers(OPT_STEP, **{k: s[k] for k in _state_names(bits)})
    return s


def _state_names(bits):
    return ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if bits == 8 else ())


def _starts(sizes, align):
    starts, off = [], 0
    for n in sizes:
        starts.append(off)
        off += -(-n // align) * align
    return starts, off


def _nearest(x):
    """Blocks of ``x`` as e4m3 values (no value but zero becomes zero) and a scale each."""
    b = x.view(-1, BLOCK)
    most = b.abs().amax(1, keepdim=True)
    code = (b * torch.where(most > 0, E4M3_MAX / most, torch.zeros_like(most))).to(torch.float8_e4m3fn).float()
    code = torch.where((code == 0) & (b != 0), torch.sign(b) * 2.0 ** -9, code)
    return code.to(torch.float8_e4m3fn).view(-1), (most / E4M3_MAX).view(-1)


# ---------------------------------------------------------------- one call
def run(state):
    return {"norm": _run_norm, "scan": _run_scan, "linear": _run_linear, "adamw": _run_adamw}[state["case"]["op"]](state)


def _run_norm(s):
    x, w, res = s["x"], s["weight"], s["residual"]
    if s["case"]["form"] == "8bit":
        if own:
            from autodist_b200.ops import functional as F
            return F.rms_norm_8bit(x, w, res, EPS)
        total, y = _plain_norm(x, w, res)
        scale = y.abs().amax(1) / E4M3_MAX
        codes = torch.where(scale[:, None] == 0, 0.0, y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        return (codes, scale) if res is None else (codes, scale, total)
    if own:
        from autodist_b200.ops import functional as F
        if res is None:
            y = F.rms_norm(x, w, eps=EPS)
            return (y,) + torch.autograd.grad(y, (x, w), s["dy"])
        y, total = F.rms_norm(x, w, res, EPS)
        return (y, total) + torch.autograd.grad((y, total), (x, w, res), (s["dy"], s["ds"]))
    with torch.no_grad():
        total, y = _plain_norm(x, w, res)
        f = total.float()
        rstd = torch.rsqrt((f * f).mean(1, keepdim=True) + EPS)
        xhat, dy = f * rstd, s["dy"].float()
        g = dy * w
        dx = rstd * (g - xhat * (g * xhat).mean(1, keepdim=True))
        dw = (dy * xhat).sum(0)
        if res is None:
            return y.to(x.dtype), dx.to(x.dtype), dw
        dx = (dx + s["ds"].float()).to(x.dtype)
        return y.to(x.dtype), total, dx, dw, dx


def _plain_norm(x, w, res):
    """The stream that leaves, and its norm. The stream is rounded to its type first: what leaves is what is normed."""
    total = x if res is None else (x.float() + res.float()).to(x.dtype)
    f = total.float()
    return total, f * torch.rsqrt((f * f).mean(1, keepdim=True) + EPS) * w


def _run_scan(s):
    x, forget, gate, state, reset = s["x"], s["forget"], s["input"], s["state"], s["reset"]
    train = s["case"]["form"] == "train"
    if own:
        from autodist_b200.ops import functional as F
        y, last = F.gated_recurrence(x, forget, gate, state=state, reset=reset)
        if not train:
            return y, last
        wanted = [t for t in (x, forget, gate, state) if t is not None]
        return (y, last) + torch.autograd.grad((y, last), wanted, (s["dy"], s["dlast"]))
    with torch.no_grad():
        f = torch.sigmoid(forget.float())
        u = torch.sigmoid(-forget.float()) if gate is None else torch.sigmoid(gate.float())
        a = f if reset is None else f.masked_fill(reset[..., None], 0.0)
        v = x.float()
        b = u * v
        b[:, 0] += a[:, 0] * state
        h = _plain_scan(a, b)
        y, last = h.to(x.dtype), h[:, -1].clone()
        if not train:
            return y, last
        # dh_t = dy_t + a_{t+1} dh_{t+1}: the same scan over reversed time
        dy = s["dy"].float()
        dy[:, -1] += s["dlast"]
        later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        dh = _plain_scan(later.flip(1), dy.flip(1)).flip(1)
        before = torch.cat([state[:, None], h[:, :-1]], 1)
        if reset is not None:
            before = before.masked_fill(reset[..., None], 0.0)
        df = dh * (before - v if gate is None else before) * f * torch.sigmoid(-forget.float())
        grads = [dh * u, df] + ([dh * v * u * torch.sigmoid(-gate.float())] if gate is not None else [])
        return (y, last) + tuple(t.to(x.dtype) for t in grads) + (a[:, 0] * dh[:, 0],)


def _plain_scan(a, b):
    """h_t = a_t h_{t-1} + b_t from zero along dimension 1, by doubling: log2(steps) passes instead of one for each step."""
    steps, reach = a.shape[1], 1
    while reach < steps:
        b = torch.cat([b[:, :reach], b[:, reach:] + a[:, reach:] * b[:, :-reach]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return b


def _run_linear(s):
    if own:
        from autodist_b200.ops import functional as F
        return F.linear_8bit(s["codes"], s["scales"], s["weight_codes"], s["weight_scales"], s["bias"])
    y = (s["codes"].float() @ s["weight_codes"].float().t()) * s["scales"][:, None] * s["weight_scales"]
    return (y if s["bias"] is None else y + s["bias"]).to(torch.bfloat16)


def _run_adamw(s):
    bits = s["case"]["bits"]
    if own:
        s["optimizer"].step()
        return dict({k: s["optimizer"].buffers[k] for k in _state_names(bits)}, values=s["values"])
    s["step"] += 1
    (b1, b2), lr = ADAMW["betas"], ADAMW["lr"]
    index, filled = s["index"], s["filled"]
    p, g = (t.float() if index is None else torch.where(filled, t[index].float(), 0.0) for t in (s["values"], s["grads"]))
    if bits == 8:
        m = (s["exp_avg"].float().view(-1, BLOCK) * s["exp_avg_scale"][:, None]).view(-1)
        v = (s["exp_avg_sq"].float().view(-1, BLOCK) * s["exp_avg_sq_scale"][:, None]).view(-1)
        v = v * v
    else:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    root = torch.sqrt(v)
    rate, spread = lr / (1 - b1 ** s["step"]), (1 - b2 ** s["step"]) ** -0.5
    p = p * (1 - lr * ADAMW["weight_decay"]) - rate * (m / (root * spread + ADAMW["eps"]))
    if index is None:
        s["values"].copy_(p)
    else:
        s["values"][index[filled]] = p[filled].to(s["values"].dtype)
    if bits == 8:
        low, high = _uniform(s["step"], p.numel())
        for name, x, u in (("exp_avg", m, low), ("exp_avg_sq", root, high)):
            codes, scale = _stochastic(x, u)
            s[name].copy_(codes)
            s[name + "_scale"].copy_(scale)
    else:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
    return dict({k: s[k] for k in _state_names(bits)}, values=s["values"])


def _mixed(seed, counter):
    """64 well-mixed bits of a counter (``counter``: int64 tensor or number; all arithmetic is modulo 2^64)."""
    def wrapped(n):
        return (n + 2 ** 63) % 2 ** 64 - 2 ** 63

    def xorshift(v, k):
        return v ^ ((v >> k) & (2 ** (64 - k) - 1))
    number = not torch.is_tensor(counter)
    v = torch.tensor([wrapped(counter)], device=DEVICE) if number else counter
    v = v * wrapped(0x9E3779B97F4A7C15) + wrapped(seed)
    v = xorshift(v, 30) * wrapped(0xBF58476D1CE4E5B9)
    v = xorshift(v, 27) * wrapped(0x94D049BB133111EB)
    v = xorshift(v, 31)
    return int(v.item()) if number else v


def _uniform(step, n):
    """Two numbers in (0, 1) for each of ``n`` places: 16 bits each of the hash that a pair of places shares."""
    words = _mixed(_mixed(OPT_SEED, step), torch.arange(n // 2, device=DEVICE))
    words = torch.stack([words & 0xFFFFFFFF, (words >> 32) & 0xFFFFFFFF], 1).view(-1)
    return (((words >> k & 0xFFFF).float() + 0.5) / 65536.0 for k in (0, 16))


def _stochastic(x, u):
    """Blocks of ``x`` as e4m3 values rounded up with the probability of what is cut off (no value but zero becomes zero), and their scales."""
    b = x.view(-1, BLOCK)
    most = b.abs().amax(1, keepdim=True)
    held = most >= TINIEST
    b = b * torch.where(held, E4M3_MAX / most, torch.zeros_like(most))
    size = b.abs()
    ulp = (size.clamp_min(2.0 ** -6).view(torch.int32) & 0x7F800000).view(torch.float32) / 8       # an eighth of the power of two below
    code = (torch.floor(size / ulp + u.view(-1, BLOCK)) * ulp).clamp_max(E4M3_MAX)
    code = torch.where((code == 0) & (size > 0), torch.full_like(code, 2.0 ** -9), code) * torch.sign(b)
    return code.to(torch.float8_e4m3fn).view(-1), torch.where(held, most / E4M3_MAX, torch.zeros_like(most)).view(-1)


# ---------------------------------------------------------------- what one call cannot do without
def work(case):
    op = case["op"]
    if op == "linear":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": m * k + n * k + 2 * m * n + 4 * (m + n * (2 if case["bias"] else 1)), "flops": 2 * m * n * k}
    if op == "adamw":
        n, size = sum(_sizes(case["hidden"], case["layers"], case["vocab"])), DTYPES[case["dtype"]].itemsize
        return {"bytes": n * (3 * size + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)), "flops": 15 * n}
    size, train = DTYPES[case["dtype"]].itemsize, case["form"] == "train"
    if op == "norm":
        n, res = case["rows"] * case["width"], case["residual"]
        moved = size * ((3 if res else 1) + (1 if train else 0))                            # x (+ residual, sum), y
        moved += size * ((4 if res else 3) if train else 0) + (0 if train else 1)            # backward: dy, (ds,) sum or x, dx; or codes
        return {"bytes": n * moved + 4 * case["width"] * (2 if train else 1) + (0 if train else 4 * case["rows"]), "flops": n * (16 if train else 8)}
    n, gates = case["batch"] * case["steps"] * case["channels"], 2 if case["input_gate"] else 1
    moved = size * (2 + gates + (1 + 2 * (1 + gates) if train else 0))
    return {"bytes": n * moved + 8 * case["batch"] * case["channels"] * (2 if train else 1) + case["batch"] * case["steps"] * case["resets"],
            "flops": n * (24 if train else 8)}


# ---------------------------------------------------------------- the same from the definitions, in 64 bits
def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return {"norm": _exact_norm, "scan": _exact_scan, "linear": _exact_linear, "adamw": _exact_adamw}[case["op"]](s)


def _exact_norm(s):
    x, w, res = s["x"].double(), s["weight"].double(), s["residual"]
    total = x if res is None else (x + res.double()).to(s["x"].dtype).double()
    norm = ((total ** 2).sum(1, keepdim=True) / x.shape[1] + EPS) ** 0.5
    y = total / norm * w
    if s["case"]["form"] == "8bit":
        scale = y.abs().max(1).values / E4M3_MAX
        return (y / scale[:, None], scale) if res is None else (y / scale[:, None], scale, total)
    g = s["dy"].double() * w
    dx = g / norm - total * (g * total).sum(1, keepdim=True) / (x.shape[1] * norm ** 3)
    dw = torch.einsum("rc,rc->c", s["dy"].double(), total / norm)
    return (y, dx, dw) if res is None else (y, total, dx + s["ds"].double(), dw, dx + s["ds"].double())


def _exact_scan(s):
    x, keep, state = s["x"].double(), 1 / (1 + torch.exp(-s["forget"].double())), s["state"].double()
    take = 1 - keep if s["input"] is None else 1 / (1 + torch.exp(-s["input"].double()))
    a = keep if s["reset"] is None else torch.where(s["reset"][..., None], 0.0, keep)
    steps = x.shape[1]
    h = torch.empty(x.shape[0], steps + 1, x.shape[2], dtype=torch.float64, device=x.device)
    h[:, 0] = state
    for t in range(steps):
        torch.addcmul(take[:, t] * x[:, t], a[:, t], h[:, t], out=h[:, t + 1])
    if s["case"]["form"] != "train":
        return h[:, 1:], h[:, -1]
    dh = s["dy"].double()
    dh[:, -1] += s["dlast"].double()
    for t in range(steps - 2, -1, -1):
        dh[:, t].addcmul_(a[:, t + 1], dh[:, t + 1])
    dforget = dh * h[:, :-1] * a * (1 - keep)
    dtake = dh * x
    grads = [dh * take, dforget - dtake * keep * (1 - keep)] if s["input"] is None else [dh * take, dforget, dtake * take * (1 - take)]
    return (h[:, 1:], h[:, -1], *grads, a[:, 0] * dh[:, 0])


def _exact_linear(s):
    y = torch.einsum("mk,nk->mn", s["codes"].double() * s["scales"].double()[:, None], s["weight_codes"].double() * s["weight_scales"].double()[:, None])
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_adamw(s):
    """The states' 8-bit values are said to be what they round: the moments over their blocks' scales."""
    case, t, (b1, b2) = s["case"], OPT_STEP + 1, ADAMW["betas"]
    sizes = _sizes(case["hidden"], case["layers"], case["vocab"])
    starts, _ = _starts(sizes, case["align"])
    places, padded = _starts(sizes, BLOCK)
    scales = {k: (s[k + "_scale"].double().repeat_interleave(BLOCK) if case["bits"] == 8 else 1.0) for k in ("exp_avg", "exp_avg_sq")}
    m, v = s["exp_avg"].double() * scales["exp_avg"], s["exp_avg_sq"].double() * scales["exp_avg_sq"]
    v = v ** 2 if case["bits"] == 8 else v
    p, g = s["values"].double(), torch.zeros(padded, dtype=torch.float64, device=DEVICE)
    spans = list(zip(starts, places, sizes))
    for o, q, n in spans:
        g[q:q + n] = s["grads"][o:o + n]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g ** 2 * (1 - b2)
    move = ADAMW["lr"] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + ADAMW["eps"])
    for o, q, n in spans:
        p[o:o + n] -= ADAMW["lr"] * ADAMW["weight_decay"] * p[o:o + n] + move[q:q + n]
    out = {"values": p, "exp_avg": m, "exp_avg_sq": v}
    if case["bits"] == 8:
        for k, x in (("exp_avg", m), ("exp_avg_sq", v ** 0.5)):
            scale = x.view(-1, BLOCK).abs().amax(1) / E4M3_MAX
            out[k], out[k + "_scale"] = torch.where(x == 0, 0.0, x / scale.repeat_interleave(BLOCK)), scale
    return out
