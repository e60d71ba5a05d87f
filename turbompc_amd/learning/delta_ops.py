"""The gated delta rule with torch autograd, under the rules of `ops`: float32 or bfloat16
tensors on one HIP device, enqueued on its current stream, states in float32."""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from .. import _lib
from .ops import (MAX_HEAD_WIDTH, MAX_HEADS, MAX_STEPS, _call, _check, _first, _ptr, _rows,
                  _step_strides, _steps, _wants_grad, _workspace)

MAX_BATCH_HEADS = 1 << 22
_DELTA = struct.Struct("@8i5P15q2Pd")  # tmpc_delta_attention, packed
assert _DELTA.size == ctypes.sizeof(_lib.DeltaAttention)


def _gate(t: torch.Tensor) -> torch.Tensor:
    """Gates (B, T, H) whose steps are less than 2^23 elements apart."""
    return t if t.shape[1] <= 1 or t.stride(1) < 1 << 23 else t.contiguous()


def _gate_strides(t: torch.Tensor) -> Tuple[int, int, int]:
    s = t.stride()
    if t.dim() == 2:
        return s[0], 0, s[1]
    return s[0], s[1] if t.shape[1] > 1 else 0, s[2]


def _delta_args(q, k, v, log_decay, beta, lengths, state, scale):
    B, T, H = log_decay.shape if log_decay.dim() == 3 else (log_decay.shape[0], 1, log_decay.shape[1])
    *_, Hv, dv = v.shape
    return _lib.DeltaAttention.from_buffer_copy(_DELTA.pack(
        B, T, H, q.shape[-2], k.shape[-2], Hv, q.shape[-1], dv, q.data_ptr(), k.data_ptr(), v.data_ptr(),
        beta.data_ptr(), log_decay.data_ptr(), *_step_strides(q), *_step_strides(k), *_step_strides(v),
        *_gate_strides(beta), *_gate_strides(log_decay), _ptr(lengths) or 0, _ptr(state) or 0, scale))


def _check_delta(q, k, v, log_decay, beta, scale, step):
    sfx = _first("q", q, (3,) if step else (4,))
    _check("k", k, q)
    _check("v", v, q)
    _check("log_decay", log_decay, q, None, torch.float32)
    *lead, Hq, dk = q.shape
    *klead, Hk, kd = k.shape if k.dim() == q.dim() else (None, 0, 0)
    *vlead, Hv, dv = v.shape if v.dim() == q.dim() else (None, 0, 0)
    *glead, H = log_decay.shape if log_decay.dim() else (None,)
    if klead != lead or kd != dk:
        raise ValueError(f"k has shape {tuple(k.shape)}, expected {(*lead, 'Hk', dk)}")
    if vlead != lead:
        raise ValueError(f"v has shape {tuple(v.shape)}, expected {(*lead, 'Hv', 'dv')}")
    if glead != lead:
        raise ValueError(f"log_decay has shape {tuple(log_decay.shape)}, expected {(*lead, 'H')}")
    _check("beta", beta, q, log_decay.shape)
    for name, n in (("q", Hq), ("k", Hk), ("v", Hv)):
        if n < 1 or H < 1 or H % n:
            raise ValueError(f"the {H} heads of log_decay are not a multiple of the {n} heads of {name}")
    if H > MAX_HEADS:
        raise ValueError(f"log_decay has {H} heads, expected at most {MAX_HEADS}")
    if lead[0] * H > MAX_BATCH_HEADS:
        raise ValueError(f"log_decay has {lead[0]} problems of {H} heads, expected at most {MAX_BATCH_HEADS} together")
    if not step and lead[1] > MAX_STEPS:
        raise ValueError(f"q has {lead[1]} steps, expected at most {MAX_STEPS}")
    for name, d in (("q and k", dk), ("v", dv)):
        if not 1 <= d <= MAX_HEAD_WIDTH:
            raise ValueError(f"{name} have heads of {d} elements, expected 1 to {MAX_HEAD_WIDTH}")
    return sfx, float(dk ** -0.5 if scale is None else scale)


def _delta_forward(q, k, v, log_decay, beta, state, lengths, scale, sfx):
    B, T, H = log_decay.shape
    dk, dv = q.shape[-1], v.shape[-1]
    o, out = q.new_empty((B, T, H, dv)), log_decay.new_empty((B, H, dk, dv))
    a = _delta_args(q, k, v, log_decay, beta, lengths, state, scale)
    nbytes, ws = _workspace("tmpc_delta_attention_workspace_bytes", q.device, q.element_size(), a, 0)
    _call(f"tmpc_delta_attention_forward_{sfx}", q.device, a, _ptr(o), _ptr(out), _ptr(ws), nbytes)
    return o, out


class _DeltaAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta, state, lengths, scale, sfx):
        ctx.save_for_backward(q, k, v, log_decay, beta, state, lengths)
        ctx.scale, ctx.sfx = scale, sfx
        ctx.set_materialize_grads(False)
        return _delta_forward(q, k, v, log_decay, beta, state, lengths, scale, sfx)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, d_out):
        q, k, v, log_decay, beta, state, lengths = ctx.saved_tensors
        # a hook may give a tensor back in another layout
        q, k, v, log_decay, beta = _steps(q), _steps(k), _steps(v), _gate(log_decay), _gate(beta)
        state = state.contiguous() if state is not None else None
        lengths = lengths.contiguous() if lengths is not None else None
        dev = q.device
        d_o = _steps(d_o) if d_o is not None else torch.zeros(log_decay.shape + v.shape[-1:], dtype=q.dtype, device=dev)
        d_out = d_out.contiguous() if d_out is not None else None
        empty = lambda t: torch.empty_like(t, memory_format=torch.contiguous_format)  # noqa: E731
        dq, dk, dv, dg, dbeta = (empty(t) for t in (q, k, v, log_decay, beta))
        d_state = empty(state) if state is not None and ctx.needs_input_grad[5] else None
        a = _delta_args(q, k, v, log_decay, beta, lengths, state, ctx.scale)
        nbytes, ws = _workspace("tmpc_delta_attention_workspace_bytes", dev, q.element_size(), a, 1)
        st = (ctypes.c_int64 * 3)(*_step_strides(d_o))
        _call(f"tmpc_delta_attention_backward_{ctx.sfx}", dev, a, _ptr(d_o), st, _ptr(d_out), _ptr(dq), _ptr(dk),
              _ptr(dv), _ptr(dg), _ptr(dbeta), _ptr(d_state), _ptr(ws), nbytes)
        return dq, dk, dv, dg, dbeta, d_state, None, None, None


def delta_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, beta: torch.Tensor,
                    state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gated delta rule over whole histories: a memory that decays by what each step says and
    that replaces what it holds under a key.

    log_decay (B, T, H) float32, <= 0 (-inf forgets everything), and beta (B, T, H); q (B, T,
    Hq, dk), k (B, T, Hk, dk), v (B, T, Hv, dv), each of Hq, Hk, Hv dividing H; T at most 2^30, widths 1 to
    128.  Per problem and head, with a_t = exp(log_decay_t),
      u_t = beta_t (v_t - a_t k_t S_{t-1}),  S_t = a_t S_{t-1} + k_t^T u_t,  o_t = scale q_t S_t,
    from state (B, H, dk, dv) float32 (zero where None), for t < lengths[b] (int32, clamped to
    0..T; None: T); later steps give zero rows, and what their inputs hold is not read.  The
    recurrence is stable for beta_t |k_t|^2 from 0 to 2: keys of unit length with beta from 0 to 1 are
    usual.  An infinite or NaN value at a live step spoils what it has a part in: no earlier step's output,
    other head or problem.  scale is dk^-1/2 where None.  Returns o (B, T, H, dv) and the state after
    each history's last step (float32).

    log_decay's gradient has the decay as a factor: it is zero where exp(log_decay) is below 2^-126, and off by
    last bits of the gradients within 256 steps of it."""
    sfx, scale = _check_delta(q, k, v, log_decay, beta, scale, False)
    B, _, H = log_decay.shape
    if state is not None:
        _check("state", state, q, (B, H, q.shape[-1], v.shape[-1]), torch.float32)
    if lengths is not None:
        _check("lengths", lengths, q, (B,), torch.int32)
    state = state.contiguous() if state is not None else None
    lengths = lengths.contiguous() if lengths is not None else None
    args = (_steps(q), _steps(k), _steps(v), _gate(log_decay), _gate(beta), state, lengths, scale, sfx)
    return _DeltaAttention.apply(*args) if _wants_grad(q, k, v, log_decay, beta, state) else _delta_forward(*args)


def delta_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                         beta: torch.Tensor, state: torch.Tensor, active: Optional[torch.Tensor] = None,
                         scale: Optional[float] = None) -> torch.Tensor:
    """One step of delta_attention for each problem: q (B, Hq, dk), k (B, Hk, dk), v (B, Hv, dv),
    log_decay and beta (B, H).  state (B, H, dk, dv), float32 and contiguous, is updated in
    place; returns o (B, H, dv).  Problems whose `active` (B,) bool is False keep their state and give
    zero.  Not differentiable."""
    sfx, scale = _check_delta(q, k, v, log_decay, beta, scale, True)
    B, H = log_decay.shape
    dv = v.shape[-1]
    _check("state", state, q, (B, H, q.shape[-1], dv), torch.float32)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    if active is not None:
        _check("active", active, q, (B,), torch.bool)
        active = active.contiguous()
    if _wants_grad(q, k, v, log_decay, beta, state):
        raise ValueError("delta_attention_step has no gradient; use delta_attention, or torch.no_grad()")
    q, k, v = _rows(q), _rows(k), _rows(v)
    o = q.new_empty((B, H, dv))
    a = _delta_args(q, k, v, log_decay, beta, None, None, scale)
    _call(f"tmpc_delta_attention_step_{sfx}", q.device, a, _ptr(active), _ptr(state), _ptr(o))
    increment_version(state)  # a backward pass that saved it has to see the change
    return o
