"""Gated recurrent language model: trained in parallel over time, answered with token by token from a state of fixed size.

A block adds its input to the residual stream and norms it, projects it to units and their forget gates, runs the gated recurrence over
time and projects back. Next to the LSTM of ``lm1b`` its gates do not depend on the state in front of them, so that a sequence is one scan
instead of a product per step. For answering, the projections' weights are kept in 8 bits and the norms hand them their rows in 8 bits.
"""
from dataclasses import dataclass

import torch
from torch import nn
import torch.nn.functional as F

from autodist_b200.ops.functional import gated_recurrence, linear, linear_8bit, quantize_rows, rms_norm, rms_norm_8bit


@dataclass
class RecurrentLMConfig:
    vocab_size: int = 30522
    width: int = 1024
    units: int = 2048
    layers: int = 18
    forget_bias: float = 2.0

    @classmethod
    def tiny(cls):
        return cls(vocab_size=200, width=64, units=96, layers=2)


class RecurrentBlock(nn.Module):
    def __init__(self, c):
        super().__init__()
        self.norm = nn.Parameter(torch.ones(c.width))
        self.w_in = nn.Parameter(torch.randn(2 * c.units, c.width) * c.width ** -0.5)      # units, then their forget gates
        self.b_in = nn.Parameter(torch.cat([torch.zeros(c.units), torch.linspace(0.0, 4.0, c.units)]))
        self.w_out = nn.Parameter(torch.randn(c.width, c.units) * (c.units * 2 * c.layers) ** -0.5)


class RecurrentLM(nn.Module):
    _autodist_leaf = True

    def __init__(self, config: RecurrentLMConfig = RecurrentLMConfig()):
        super().__init__()
        c = self.config = config
        self.emb = nn.Parameter(torch.randn(c.vocab_size, c.width) * 0.02)
        self.blocks = nn.ModuleList(RecurrentBlock(c) for _ in range(c.layers))
        self.norm = nn.Parameter(torch.ones(c.width))
        self.w_vocab = nn.Parameter(torch.randn(c.vocab_size, c.width) * c.width ** -0.5)

    def features(self, tokens, states=None, reset=None):
        """Normed outputs ``[B, T, width]`` and every block's last state, from ``states`` (zeros without any)."""
        c = self.config
        stream = F.embedding(tokens, self.emb).to(torch.bfloat16 if tokens.is_cuda else torch.float32)
        out, last = None, []
        for k, b in enumerate(self.blocks):
            if out is None:
                y = rms_norm(stream, b.norm)
            else:
                y, stream = rms_norm(out, b.norm, stream)
            x, forget = linear(y, b.w_in, b.b_in).chunk(2, -1)
            h, state = gated_recurrence(x, forget, state=None if states is None else states[k], reset=reset, forget_bias=c.forget_bias)
            last.append(state)
            out = linear(h, b.w_out)
        return rms_norm(out, self.norm, stream)[0], last

    def forward(self, x, y):
        """Mean cross-entropy of the next tokens ``y`` after ``x``, int64 ``[batch, steps]``."""
        features, _ = self.features(x)
        return F.cross_entropy(linear(features, self.w_vocab).flatten(0, 1).float(), y.flatten())

    @torch.no_grad()
    def answerer(self):
        """The model with its projections in 8 bits, for answering."""
        return EightBitAnswerer(self)


class EightBitAnswerer:
    """Logits from weights in 8 bits: prompts and single tokens go the same way."""

    def __init__(self, model):
        self.model = model
        self.projections = [(quantize_rows(b.w_in.detach().float()), b.b_in.detach().float(), quantize_rows(b.w_out.detach().float())) for b in model.blocks]
        self.vocab = quantize_rows(model.w_vocab.detach().float())

    @torch.no_grad()
    def __call__(self, tokens, states=None):
        """Logits ``[B, vocab]`` after the last of ``tokens`` [B, T], and the states to go on from."""
        m, c = self.model, self.model.config
        stream = F.embedding(tokens, m.emb).to(torch.bfloat16)
        out, last = None, []
        for k, (b, (w_in, b_in, w_out)) in enumerate(zip(m.blocks, self.projections)):
            if out is None:
                rows = rms_norm_8bit(stream, b.norm)
            else:
                *rows, stream = rms_norm_8bit(out, b.norm, stream)
            x, forget = linear_8bit(*rows, *w_in, b_in).chunk(2, -1)
            h, state = gated_recurrence(x, forget, state=None if states is None else states[k], forget_bias=c.forget_bias)
            last.append(state)
            out = linear_8bit(*quantize_rows(h), *w_out)
        codes, scales, _ = rms_norm_8bit(out[:, -1], m.norm, stream[:, -1])
        return linear_8bit(codes, scales, *self.vocab), last


def cyclic_tokens(batch, steps, vocab, period=7, seed=0):
    """Token sequences that repeat with ``period``, each from a start of its own: what comes next can be learned (synthetic)."""
    g = torch.Generator().manual_seed(seed)
    words = torch.randint(0, vocab, (period,), generator=g)
    at = torch.randint(0, period, (batch, 1), generator=g) + torch.arange(steps + 1)
    ids = words[at % period]
    return {"x": ids[:, :-1].contiguous(), "y": ids[:, 1:].contiguous()}
