"""Optimizers with state layouts of their own."""
import torch

from autodist_b200 import ops

#: Elements of a parameter that share a scale of the 8-bit moments.
BLOCK = 256
E4M3_MAX = 448.0
#: Blocks whose largest moment is smaller are held as zeros: the inverse of their scale would overflow.
TINIEST = 2.0 ** -100


def _round_up(n, m):
    return (n + m - 1) // m * m


def _wrapped(n):
    """``n`` modulo 2^64 as an int64."""
    return (n + 2 ** 63) % 2 ** 64 - 2 ** 63


def _mixed(seed, counter):
    """64 mixed bits of each counter (int64 tensor), as the kernel draws them."""
    def xorshift(v, k):
        return v ^ ((v >> k) & (2 ** (64 - k) - 1))
    v = counter * _wrapped(0x9E3779B97F4A7C15) + _wrapped(seed)
    v = xorshift(v, 30) * _wrapped(0xBF58476D1CE4E5B9)
    v = xorshift(v, 27) * _wrapped(0x94D049BB133111EB)
    return xorshift(v, 31)


def _scales(blocks):
    """What turns blocks into sizes of at most 448, and back, in the kernel's roundings."""
    most = blocks.abs().amax(1, keepdim=True)
    held = ~(most < TINIEST)
    return torch.where(held, most.reciprocal() * E4M3_MAX, 0.0), torch.where(held, most * (1.0 / E4M3_MAX), 0.0)


def _codes(x, u):
    """``(codes, scales)`` of ``x`` in blocks. ``u`` in (0, 1): a size is rounded up where it and what is cut off add up to one; nothing but zero
    becomes zero. Without ``u``: rounded to the nearest."""
    b = x.view(-1, BLOCK)
    inverse, scale = _scales(b)
    size = (b * inverse).abs()
    ulp = (size.clamp_min(2.0 ** -6).view(torch.int32) & 0x7F800000).view(torch.float32) / 8
    code = (torch.floor(size / ulp + (0.5 if u is None else u.view(-1, BLOCK))) * ulp).clamp_max(E4M3_MAX)
    code = torch.where((code == 0) & (size > 0), 2.0 ** -9, code)
    return torch.copysign(code, b).to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _values(codes, scale):
    return (codes.float().view(-1, BLOCK) * scale[:, None]).view(-1)


class ListAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) that updates all parameters of a group in one launch, moments in fp32 or in 8 bits.

    With ``state_bits=8`` every 256 elements of a parameter share an fp32 scale (the largest size over 448); the first moment and the root
    of the second are ``float8_e4m3fn`` values in it, rounded up or down at random with the probability of what is cut off: a step changes
    the second moment by a thousandth, which rounding to the nearest would undo. The random bits are a hash of ``seed``, the step and the
    element's place, so that a step can be repeated. The update itself uses the moments before they are rounded. 2 bytes (and 1/32) per
    parameter instead of 8. A gradient that is not finite spoils the moments of its block.

    Parameters and gradients are bf16 or fp32. The steps taken are counted per group in device memory (``torch.cuda.graph`` replays follow
    it); ``lr`` may be an fp32 tensor of one element on the GPU. Parameters without a gradient are left as they are. On CPU tensors
    the same arithmetic runs as PyTorch expressions."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=8, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"ListAdamW: moments in 8 or in 32 bits, got {state_bits}")
        if not torch.is_tensor(lr) and not lr >= 0:
            raise ValueError(f"ListAdamW: bad learning rate {lr}")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError(f"ListAdamW: bad betas {betas}")
        if not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"ListAdamW: bad eps {eps} or weight decay {weight_decay}")
        self.state_bits, self.seed = state_bits, int(seed)
        self._groups = []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed))

    # ------------------------------------------------------------------ state
    def _names(self):
        return ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if self.state_bits == 8 else ())

    def _group(self, index):
        """The moments of a group: flat buffers in which every parameter starts on a block, made when they are first needed."""
        while len(self._groups) <= index:
            self._groups.append(None)
        params = self.param_groups[index]["params"]
        own = self._groups[index]
        if own is not None and len(own["params"]) == len(params) and own["buffers"]["exp_avg"].device == params[0].device:
            return own
        for p in params:
            if p.dtype not in (torch.bfloat16, torch.float32):
                raise TypeError(f"ListAdamW: bf16 or fp32 parameters needed, got {p.dtype}")
            if p.device != params[0].device:
                raise ValueError("ListAdamW: the parameters of a group must be on one device")
        places, total = [], 0
        for p in params:
            places.append(total)
            total += _round_up(p.numel(), BLOCK)
        dev, bits8 = params[0].device, self.state_bits == 8
        kind = torch.float8_e4m3fn if bits8 else torch.float32
        buffers = {k: torch.zeros(total, dtype=kind, device=dev) for k in ("exp_avg", "exp_avg_sq")}
        if bits8:
            buffers.update({k: torch.zeros(total // BLOCK, dtype=torch.float32, device=dev) for k in ("exp_avg_scale", "exp_avg_sq_scale")})
        # steps taken, and a word in which the kernel's blocks count themselves
        own = self._groups[index] = {"params": list(params), "places": places, "buffers": buffers, "step": torch.zeros(2, dtype=torch.int64, device=dev)}
        if dev.type == "cuda" and total:
            own["list"] = ops.ext(required=True).adamw_list(own["params"], places, buffers["exp_avg"], buffers["exp_avg_sq"], buffers.get("exp_avg_scale"),
                                                            buffers.get("exp_avg_sq_scale"), own["step"], self.seed + index)
            views = ops.ext(required=True).adamw_views(own["list"])
        else:
            views = [[b[o:o + p.numel()].view(p.shape) if b.numel() == total else b[o // BLOCK:(o + _round_up(p.numel(), BLOCK)) // BLOCK] for b in buffers.values()]
                     for p, o in zip(params, places)]
        taken = own["step"][:1]
        for p, v in zip(params, views):
            self.state[p] = dict(zip(buffers, v), step=taken)
        return own

    @property
    def buffers(self):
        """The flat moments of the only group, by name."""
        if len(self.param_groups) != 1:
            raise ValueError("ListAdamW: buffers of several groups are in their parameters' states")
        return self._group(0)["buffers"]

    def load_buffers(self, step, **buffers):
        """Copies flat moments, as ``buffers`` names them, of the only group, which has taken ``step`` steps."""
        own = self.buffers
        if set(buffers) != set(own):
            raise ValueError(f"ListAdamW: {sorted(own)} needed, got {sorted(buffers)}")
        for k, b in buffers.items():
            if b.shape != own[k].shape or b.dtype != own[k].dtype:
                raise ValueError(f"ListAdamW: {k} is {tuple(own[k].shape)} {own[k].dtype}, got {tuple(b.shape)} {b.dtype}")
            own[k].copy_(b)
        self._group(0)["step"].copy_(torch.tensor([step, 0]))

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for index, group in enumerate(self.param_groups):
            if not group["params"]:
                continue
            own = self._group(index)
            if "list" in own:
                lr, (b1, b2) = group["lr"], group["betas"]
                on_gpu = torch.is_tensor(lr) and lr.is_cuda
                ops.ext(required=True).adamw_list_step(own["list"], 0.0 if on_gpu else float(lr), lr if on_gpu else None, b1, b2, group["eps"],
                                                       group["weight_decay"])
            else:
                self._step_plain(own, group)
        return loss

    def _step_plain(self, own, group):
        live = [(p, o) for p, o in zip(own["params"], own["places"]) if p.grad is not None and p.numel()]
        if not live:
            return
        own["step"][0] += 1
        t, lr, (b1, b2) = int(own["step"][0]), float(group["lr"]), group["betas"]
        key = int(_mixed(self.seed + self._groups.index(own), torch.tensor([t]))[0])
        rate, spread = lr / (1 - b1 ** t), (1 - b2 ** t) ** -0.5
        buffers = own["buffers"]
        for p, o in live:
            if p.grad.is_sparse:
                raise RuntimeError("ListAdamW: sparse gradients are not supported")
            n, padded = p.numel(), _round_up(p.numel(), BLOCK)
            at, blocks = slice(o, o + padded), slice(o // BLOCK, (o + padded) // BLOCK)
            w, g = (torch.nn.functional.pad(v.detach().float().reshape(-1), (0, padded - n)) for v in (p, p.grad))
            m, v = buffers["exp_avg"][at], buffers["exp_avg_sq"][at]
            if self.state_bits == 8:
                m, v = _values(m, buffers["exp_avg_scale"][blocks]), _values(v, buffers["exp_avg_sq_scale"][blocks]).square()
            m = b1 * m + (1 - b1) * g
            v = b2 * v + (1 - b2) * (g * g)
            root = v.sqrt()
            w = w * (1 - lr * group["weight_decay"]) - rate * (m / (root * spread + group["eps"]))
            p.copy_(w[:n].view(p.shape))
            if self.state_bits == 8:
                bits = _mixed(key, torch.arange(o // 2, (o + padded) // 2, device=p.device))
                bits = torch.stack([bits & 0xFFFFFFFF, (bits >> 32) & 0xFFFFFFFF], 1).view(-1)
                for name, x, shift in (("exp_avg", m, 0), ("exp_avg_sq", root, 16)):
                    codes, scale = _codes(x, ((bits >> shift & 0xFFFF).float() + 0.5) / 65536.0)
                    buffers[name][at].copy_(codes)
                    buffers[name + "_scale"][blocks].copy_(scale)
            else:
                buffers["exp_avg"][at].copy_(m)
                buffers["exp_avg_sq"][at].copy_(v)

    # ------------------------------------------------------------------ checkpoints
    def slots_of(self, p):
        """The moments of a parameter in fp32 and in its shape, by ``torch.optim.AdamW``'s names, and its group's steps; ``None`` before the first step."""
        if p not in self.state:
            return None
        st, n = self.state[p], p.numel()
        out = {"step": float(st["step"][0])}
        for k in ("exp_avg", "exp_avg_sq"):
            x = st[k].float()
            if self.state_bits == 8:
                flat = torch.nn.functional.pad(x.reshape(-1), (0, _round_up(n, BLOCK) - n))
                x = _values(flat, st[k + "_scale"])[:n].view(p.shape)
                x = x.square() if k == "exp_avg_sq" else x
            out[k] = x
        return out

    def load_slots(self, p, slots, step):
        """The counterpart of ``slots_of``; 8-bit moments are rounded to the nearest."""
        index = next(i for i, g in enumerate(self.param_groups) if any(q is p for q in g["params"]))
        own = self._group(index)
        for k in ("exp_avg", "exp_avg_sq"):
            if k not in slots:
                continue
            x = slots[k].detach().to(device=p.device, dtype=torch.float32)
            if self.state_bits == 8:
                x = x.sqrt() if k == "exp_avg_sq" else x
                flat = torch.nn.functional.pad(x.reshape(-1), (0, _round_up(p.numel(), BLOCK) - p.numel()))
                codes, scale = _codes(flat, None)
                self.state[p][k].copy_(codes[:p.numel()].view(p.shape))
                self.state[p][k + "_scale"].copy_(scale)
            else:
                self.state[p][k].copy_(x.view(p.shape))
        own["step"].copy_(torch.tensor([int(step), 0]))

    def state_dict(self):
        for index, group in enumerate(self.param_groups):
            if group["params"]:
                self._group(index)
        return super().state_dict()

    def load_state_dict(self, state_dict):
        """Restores what ``state_dict`` gave: values and scales are copied as they are."""
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("ListAdamW: the state is of other parameter groups")
        if any(g["state_bits"] != self.state_bits for g in groups):
            raise ValueError(f"ListAdamW: the state's moments are not in {self.state_bits} bits")
        for index, (group, saved) in enumerate(zip(self.param_groups, groups)):
            if group["params"]:
                self._group(index)
            for p, key in zip(group["params"], saved["params"]):
                for k, v in state_dict["state"].get(key, {}).items():
                    self.state[p][k].copy_(v)
            group.update({k: v for k, v in saved.items() if k != "params"})
