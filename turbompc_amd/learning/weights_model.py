"""A history model for tracking weights: what a problem's vehicle has seen in, the
weights of its differentiable solve out.

Each step of a history (B, T, features) is projected to a residual stream; a
block is norm -> memory -> norm -> gated feed-forward, each adding to
the stream inside the next norm; the memory is linear attention with a decay per head, or the
gated delta rule, whose decays and rates are read from each step; the last live step's row
gives, per problem, positive weights for the keys and sizes asked for (those of
`TurboMPCSolver.get_differentiable_solve_function`, whose gradients flow back into
the model).  Training runs whole ragged histories (`forward`); a control loop
adds one step per period (`step`), its memory being one fp32 state per layer,
whatever the history's length.  The plain products (projections in and out) are
torch's.
"""
from __future__ import annotations

from typing import Dict, List, NamedTuple, Optional

import torch
from torch import nn

from . import delta_ops, norm_ops, ops


class HistoryState(NamedTuple):
    """What `step` carries from period to period."""
    layers: List[torch.Tensor]  # (B, heads, d, d) float32 each


def _norm(a, s, weight, bias, p=0.0, key=None, call=0):
    """(norm of the stream, the stream): the stream is d(a) + s, d dropping elements with probability p."""
    if bias is not None:
        return norm_ops.layer_norm_residual(a, s, weight, bias, dropout=p, key=key, call=call)
    return ops.rms_norm_residual(norm_ops.dropout(a, p, key, call) if p > 0.0 else a, s, weight)


class _Block(nn.Module):
    def __init__(self, width: int, heads: int, kv_heads: int, hidden: int, memory: str, norm: str, kw):
        super().__init__()
        self.heads, self.kv_heads, self.d = heads, kv_heads, width // heads
        linear = lambda o, i: nn.Parameter(torch.randn(o, i, **kw) * i ** -0.5)  # noqa: E731
        self.norm_attention = nn.Parameter(torch.ones(width, **kw))
        self.norm_ff = nn.Parameter(torch.ones(width, **kw))
        self.w_qkv = linear((heads + 2 * kv_heads) * self.d, width)
        self.w_out = linear(width, width)
        self.w_gate, self.w_up, self.w_down = linear(hidden, width), linear(hidden, width), linear(width, hidden)
        # a head's memory halves after 1 to 128 steps
        decay = -0.6931472 * torch.exp2(-torch.linspace(0.0, 7.0, heads, device=kw.get("device")))
        if memory == "delta":  # as it is read from a step that says nothing; the softplus' argument
            self.w_gates = nn.Parameter(0.1 * torch.randn(2 * heads, width, **kw) * width ** -0.5)
            self.decay_bias = nn.Parameter(torch.log(torch.expm1(-decay)).to(kw["dtype"]))
        else:
            self.register_buffer("log_decay", decay)
        if norm == "layer":
            self.norm_attention_bias = nn.Parameter(torch.zeros(width, **kw))
            self.norm_ff_bias = nn.Parameter(torch.zeros(width, **kw))

    def _apply(self, fn, *args, **kwargs):
        # a cast of the model is one of its parameters: the operator takes float32 decays
        decay = getattr(self, "log_decay", None)
        super()._apply(fn, *args, **kwargs)
        if decay is not None and self.log_decay.dtype != decay.dtype:
            self.log_decay = decay.to(self.log_decay.device)
        return self

    def qkv(self, y):
        x = nn.functional.linear(y, self.w_qkv).unflatten(-1, (-1, self.d))
        return x.split([self.heads, self.kv_heads, self.kv_heads], dim=-2)

    def delta(self, y):
        """The delta rule's arguments: keys of unit length, decays in float32 and rates in 0 .. 1."""
        q, k, v = self.qkv(y)
        k = nn.functional.normalize(k.float(), dim=-1).to(k.dtype)
        decay, rate = nn.functional.linear(y, self.w_gates).split(self.heads, dim=-1)
        return q, k, v, -nn.functional.softplus(decay.float() + self.decay_bias.float()), torch.sigmoid(rate)

    def attend(self, y, lengths):
        if hasattr(self, "w_gates"):
            return delta_ops.delta_attention(*self.delta(y), lengths=lengths)[0]
        return ops.decay_attention(*self.qkv(y), self.log_decay, lengths=lengths)[0]

    def attend_step(self, y, memory, active):
        if hasattr(self, "w_gates"):
            return delta_ops.delta_attention_step(*self.delta(y), memory, active=active)
        return ops.decay_attention_step(*self.qkv(y), self.log_decay, memory, active=active)

    def norm(self, name, a, s, drop=(0.0, None, 0)):
        return _norm(a, s, getattr(self, name), getattr(self, name + "_bias", None), *drop)

    def finish(self, o, s, drop=(0.0, None, 0)):
        """(the block's addition to the stream, the stream before it)."""
        a = nn.functional.linear(o.flatten(-2), self.w_out)
        y, s = self.norm("norm_ff", a, s, drop)
        return ops.gated_feed_forward(y, self.w_gate, self.w_up, self.w_down), s


class HistoryWeights(nn.Module):
    """sizes: {weight key: number of weights}, e.g. {"weights_penalization_reference_state_trajectory": nx}.
    memory: "decay" or "delta"; norm: "rms" or "layer"; dropout: of every block's additions to the stream,
    while training."""

    def __init__(self, features: int, sizes: Dict[str, int], width: int = 128, layers: int = 2, heads: int = 4,
                 kv_heads: Optional[int] = None, hidden: Optional[int] = None, floor: float = 1e-3,
                 dtype: torch.dtype = torch.float32, device="cuda", memory: str = "decay", norm: str = "rms",
                 dropout: float = 0.0):
        super().__init__()
        if width % heads:
            raise ValueError(f"the width {width} is not a multiple of the {heads} heads")
        if memory not in ("decay", "delta") or norm not in ("rms", "layer"):
            raise ValueError(f"unknown memory {memory!r} or norm {norm!r}; use decay or delta, rms or layer")
        if not 0.0 <= dropout < 1.0:
            raise ValueError(f"dropout must be at least 0 and less than 1, got {dropout}")
        kw = dict(dtype=dtype, device=device)
        self.sizes, self.floor, self.dropout = dict(sizes), float(floor), float(dropout)
        self.w_in = nn.Parameter(torch.randn(width, features, **kw) * features ** -0.5)
        self.blocks = nn.ModuleList(_Block(width, heads, kv_heads or heads, hidden or 4 * width, memory, norm, kw)
                                    for _ in range(layers))
        self.norm_out = nn.Parameter(torch.ones(width, **kw))
        if norm == "layer":
            self.norm_out_bias = nn.Parameter(torch.zeros(width, **kw))
        self.w_heads = nn.Parameter(torch.zeros(sum(self.sizes.values()), width, **kw))
        self.bias = nn.Parameter(torch.full((sum(self.sizes.values()),), 0.5413, **kw))  # softplus: 1

    def _weights(self, y) -> Dict[str, torch.Tensor]:
        w = nn.functional.softplus(nn.functional.linear(y, self.w_heads, self.bias).float()) + self.floor
        return dict(zip(self.sizes, w.split(list(self.sizes.values()), dim=-1)))

    def forward(self, history: torch.Tensor, lengths: Optional[torch.Tensor] = None,
                key: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """Weights (B, size) from histories (B, T >= 1, features); lengths (B,) int32 of ragged
        ones, clamped to 0..T (a problem without history is read from its first row's stream
        alone).  A model with dropout needs the step's key while it trains (`dropout`'s: an int64 tensor
        (seed, step), step advanced after the backward pass)."""
        p = self.dropout if self.training else 0.0
        if p > 0.0 and key is None:
            raise ValueError("a model with dropout needs a key while it trains: an int64 tensor (seed, step)")
        B, T = history.shape[:2]
        if T < 1:
            raise ValueError("the histories have no rows")
        x = history.to(self.w_in.dtype)
        if lengths is not None:
            lengths = lengths.clamp(0, T)
            # rows past a history's end may hold anything, which w_in's gradient would read
            live = torch.arange(T, device=x.device) < lengths[:, None]
            x = torch.where(live[..., None], x, torch.zeros((), dtype=x.dtype, device=x.device))
        a, s = nn.functional.linear(x, self.w_in), None
        for i, b in enumerate(self.blocks):  # the projection of the rows, which comes first, is never dropped
            y, s = b.norm("norm_attention", a, s, (p if i else 0.0, key, 2 * i))
            a, s = b.finish(b.attend(y, lengths), s, (p, key, 2 * i + 1))
        at = torch.full((B,), T, device=a.device) if lengths is None else lengths
        at = (at.long() - 1).clamp(min=0)[:, None, None].expand(-1, -1, a.shape[-1])
        y, _ = _norm(a.gather(1, at)[:, 0], s.gather(1, at)[:, 0], self.norm_out, getattr(self, "norm_out_bias", None), p, key,
                     2 * len(self.blocks))
        return self._weights(y)

    def initial_state(self, B: int) -> HistoryState:
        return HistoryState([torch.zeros((B, b.heads, b.d, b.d), dtype=torch.float32, device=b.w_qkv.device)
                             for b in self.blocks])

    @torch.no_grad()
    def step(self, row: torch.Tensor, state: HistoryState, active: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """Weights (B, size) after one more row (B, features) of every problem whose `active` (B,)
        bool is True; the state is updated in place."""
        a, s = nn.functional.linear(row.to(self.w_in.dtype), self.w_in), None
        for b, memory in zip(self.blocks, state.layers):
            y, s = b.norm("norm_attention", a, s)
            a, s = b.finish(b.attend_step(y, memory, active), s)
        y, _ = _norm(a, s, self.norm_out, getattr(self, "norm_out_bias", None))
        return self._weights(y)
