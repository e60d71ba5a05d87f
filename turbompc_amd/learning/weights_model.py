"""A history model for tracking weights: what a problem's vehicle has seen in, the
weights of its differentiable solve out.

Each step of a history (B, T, features) is projected to a residual stream; a
block is norm -> decay attention -> norm -> gated feed-forward, each adding to
the stream inside the next norm; the last live step's row gives, per problem,
positive weights for the keys and sizes asked for (those of
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

from . import ops


class HistoryState(NamedTuple):
    """What `step` carries from period to period."""
    layers: List[torch.Tensor]  # (B, heads, d, d) float32 each


class _Block(nn.Module):
    def __init__(self, width: int, heads: int, kv_heads: int, hidden: int, kw):
        super().__init__()
        self.heads, self.kv_heads, self.d = heads, kv_heads, width // heads
        linear = lambda o, i: nn.Parameter(torch.randn(o, i, **kw) * i ** -0.5)  # noqa: E731
        self.norm_attention = nn.Parameter(torch.ones(width, **kw))
        self.norm_ff = nn.Parameter(torch.ones(width, **kw))
        self.w_qkv = linear((heads + 2 * kv_heads) * self.d, width)
        self.w_out = linear(width, width)
        self.w_gate, self.w_up, self.w_down = linear(hidden, width), linear(hidden, width), linear(width, hidden)
        # a head's memory halves after 1 to 128 steps
        self.register_buffer("log_decay", -0.6931472 * torch.exp2(-torch.linspace(0.0, 7.0, heads, device=kw.get("device"))))

    def _apply(self, fn, *args, **kwargs):
        # a cast of the model is one of its parameters: the operator takes float32 decays
        decay = self.log_decay
        super()._apply(fn, *args, **kwargs)
        if self.log_decay.dtype != decay.dtype:
            self.log_decay = decay.to(self.log_decay.device)
        return self

    def qkv(self, y):
        x = nn.functional.linear(y, self.w_qkv).unflatten(-1, (-1, self.d))
        return x.split([self.heads, self.kv_heads, self.kv_heads], dim=-2)

    def finish(self, o, s):
        """(the block's addition to the stream, the stream before it)."""
        a = nn.functional.linear(o.flatten(-2), self.w_out)
        y, s = ops.rms_norm_residual(a, s, self.norm_ff)
        return ops.gated_feed_forward(y, self.w_gate, self.w_up, self.w_down), s


class HistoryWeights(nn.Module):
    """sizes: {weight key: number of weights}, e.g. {"weights_penalization_reference_state_trajectory": nx}."""

    def __init__(self, features: int, sizes: Dict[str, int], width: int = 128, layers: int = 2, heads: int = 4,
                 kv_heads: Optional[int] = None, hidden: Optional[int] = None, floor: float = 1e-3,
                 dtype: torch.dtype = torch.float32, device="cuda"):
        super().__init__()
        if width % heads:
            raise ValueError(f"the width {width} is not a multiple of the {heads} heads")
        kw = dict(dtype=dtype, device=device)
        self.sizes, self.floor = dict(sizes), float(floor)
        self.w_in = nn.Parameter(torch.randn(width, features, **kw) * features ** -0.5)
        self.blocks = nn.ModuleList(_Block(width, heads, kv_heads or heads, hidden or 4 * width, kw) for _ in range(layers))
        self.norm_out = nn.Parameter(torch.ones(width, **kw))
        self.w_heads = nn.Parameter(torch.zeros(sum(self.sizes.values()), width, **kw))
        self.bias = nn.Parameter(torch.full((sum(self.sizes.values()),), 0.5413, **kw))  # softplus: 1

    def _weights(self, y) -> Dict[str, torch.Tensor]:
        w = nn.functional.softplus(nn.functional.linear(y, self.w_heads, self.bias).float()) + self.floor
        return dict(zip(self.sizes, w.split(list(self.sizes.values()), dim=-1)))

    def forward(self, history: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """Weights (B, size) from histories (B, T >= 1, features); lengths (B,) int32 of ragged
        ones, clamped to 0..T (a problem without history is read from its first row's stream
        alone)."""
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
        for b in self.blocks:
            y, s = ops.rms_norm_residual(a, s, b.norm_attention)
            o, _ = ops.decay_attention(*b.qkv(y), b.log_decay, lengths=lengths)
            a, s = b.finish(o, s)
        at = torch.full((B,), T, device=a.device) if lengths is None else lengths
        at = (at.long() - 1).clamp(min=0)[:, None, None].expand(-1, -1, a.shape[-1])
        y, _ = ops.rms_norm_residual(a.gather(1, at)[:, 0], s.gather(1, at)[:, 0], self.norm_out)
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
            y, s = ops.rms_norm_residual(a, s, b.norm_attention)
            o = ops.decay_attention_step(*b.qkv(y), b.log_decay, memory, active=active)
            a, s = b.finish(o, s)
        y, _ = ops.rms_norm_residual(a, s, self.norm_out)
        return self._weights(y)
