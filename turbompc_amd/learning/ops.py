"""The history model's operators with torch autograd.

Data are float32 or bfloat16 tensors on one HIP device (the parameters of a call
in the same type); states and statistics are float32.  Every call is enqueued on
`torch.cuda.current_stream()` of that device and waits for nothing.  Rows (the
last axis) are read in place when contiguous, whatever the other strides, and
copied otherwise.  Shapes, types and devices that a kernel does not take raise
ValueError or TypeError before anything is enqueued; a failure in the library
raises TmpcError.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib

_SUFFIX = {torch.float32: "f32", torch.bfloat16: "bf16"}
_ACTIVATIONS = {"silu": 0, "gelu": 1}
MAX_HEAD_WIDTH = 128
MAX_NORM_WIDTH = 8192


def _suffix(dtype: torch.dtype) -> str:
    if dtype not in _SUFFIX:
        raise TypeError(f"unsupported dtype {dtype}; use float32 or bfloat16")
    return _SUFFIX[dtype]


def _check(name: str, t: torch.Tensor, like: torch.Tensor, shape=None, dtype=None):
    """t as given, with like's device and `dtype` (like's) and `shape`."""
    if not torch.is_tensor(t):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    dtype = like.dtype if dtype is None else dtype
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def _first(name: str, t: torch.Tensor, dims) -> str:
    """The suffix of the call whose first argument is t."""
    if not torch.is_tensor(t):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    sfx = _suffix(t.dtype)
    if t.device.type != "cuda":
        raise ValueError(f"{name} is on {t.device}; the operators run on a HIP device")
    if t.dim() not in dims:
        raise ValueError(f"{name} has {t.dim()} dimensions, expected {' or '.join(map(str, dims))}")
    return sfx


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous rows: itself where it has them."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _matrix(t: torch.Tensor) -> torch.Tensor:
    """t as (rows, last axis) with contiguous rows: a view where one exists."""
    return _rows(t.reshape(-1, t.shape[-1]))


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return t.data_ptr() if t is not None and t.numel() else None


def _call(fn: str, device: torch.device, *args):
    with torch.cuda.device(device):
        _lib.check(fn, getattr(_lib.load(), fn)(_lib.stream_handle(device), *args))


# ------------------------------------------------------------------ norm --
class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, sfx, train):
        xm = _matrix(x)
        rm = _matrix(residual) if residual is not None else None
        w = weight.contiguous()
        M, D = xm.shape
        y, s = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(x.shape, dtype=x.dtype, device=x.device)
        rstd = torch.empty(M, dtype=torch.float32, device=x.device) if train else None
        _call(f"tmpc_rms_norm_forward_{sfx}", x.device, M, D, _ptr(xm), xm.stride(0), _ptr(rm),
              rm.stride(0) if rm is not None else 0, _ptr(w), eps, _ptr(y), _ptr(s), _ptr(rstd))
        ctx.sfx, ctx.has_residual = sfx, residual is not None
        if train:
            ctx.save_for_backward(s, w, rstd)
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds):
        s, w, rstd = ctx.saved_tensors
        D = s.shape[-1]
        M = s.numel() // D
        dym = _matrix(dy) if dy is not None else torch.zeros((M, D), dtype=s.dtype, device=s.device)
        dsm = _matrix(ds) if ds is not None else None
        dx, dw = torch.empty_like(s), torch.empty_like(w)
        nbytes = _lib.load().tmpc_rms_norm_backward_workspace_bytes(s.element_size(), M, D)
        ws = _lib.workspace(nbytes, s.device)
        _call(f"tmpc_rms_norm_backward_{ctx.sfx}", s.device, M, D, _ptr(dym), dym.stride(0), _ptr(dsm),
              dsm.stride(0) if dsm is not None else 0, _ptr(s), D, _ptr(w), _ptr(rstd), _ptr(dx), _ptr(dw), _ptr(ws),
              nbytes)
        return dx, dx if ctx.has_residual else None, dw, None, None, None


def rms_norm_residual(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                      eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, s): s = x + residual (x where residual is None) and
    y = s / sqrt(mean(s^2) + eps) * weight over the last axis (at most 8192 wide).
    y is formed from the unrounded sum."""
    sfx = _first("x", x, range(1, 9))
    D = x.shape[-1]
    if not 1 <= D <= MAX_NORM_WIDTH:
        raise ValueError(f"x has rows of {D} elements, expected 1 to {MAX_NORM_WIDTH}")
    if residual is not None:
        _check("residual", residual, x, x.shape)
    _check("weight", weight, x, (D,))
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight))
    return _RmsNorm.apply(x, residual, weight, float(eps), sfx, train)


# ------------------------------------------------------------- attention --
def _attention_args(q, k, v, log_decay, lengths, state, scale, step=False):
    B, H, dk = q.shape[0], q.shape[-2], q.shape[-1]
    T = 1 if step else q.shape[1]
    a = _lib.DecayAttention(B=B, T=T, H=H, Hk=k.shape[-2], dk=dk, dv=v.shape[-1], q=_ptr(q), k=_ptr(k), v=_ptr(v),
                            log_decay=_ptr(log_decay), lengths=_ptr(lengths), state_in=_ptr(state), scale=scale)
    for name, t in (("q_stride", q), ("k_stride", k), ("v_stride", v)):
        st = t.stride()
        setattr(a, name, (ctypes.c_int64 * 3)(st[0], 0 if step else st[1], st[-2]))
    return a


def _check_attention(q, k, v, log_decay, scale, step):
    sfx = _first("q", q, (3,) if step else (4,))
    lead = tuple(q.shape[:-2])
    H, dk = q.shape[-2:]
    _check("k", k, q)
    _check("v", v, q)
    if k.dim() != q.dim() or tuple(k.shape[:-2]) != lead or k.shape[-1] != dk:
        raise ValueError(f"k has shape {tuple(k.shape)}, expected {lead + ('Hk', dk)}")
    Hk = k.shape[-2]
    if v.dim() != q.dim() or tuple(v.shape[:-1]) != lead + (Hk,):
        raise ValueError(f"v has shape {tuple(v.shape)}, expected {lead + (Hk, 'dv')}")
    if H < 1 or Hk < 1 or H % Hk:
        raise ValueError(f"the {H} heads of q are not a multiple of the {Hk} heads of k and v")
    for name, d in (("q and k", dk), ("v", v.shape[-1])):
        if not 1 <= d <= MAX_HEAD_WIDTH:
            raise ValueError(f"{name} have heads of {d} elements, expected 1 to {MAX_HEAD_WIDTH}")
    _check("log_decay", log_decay, q, (H,), torch.float32)
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant of the model: it takes no gradient")
    return sfx, float(dk ** -0.5 if scale is None else scale)


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale, sfx, train):
        q, k, v = _rows(q), _rows(k), _rows(v)
        log_decay = log_decay.contiguous()
        state = state.contiguous() if state is not None else None
        lengths = lengths.contiguous() if lengths is not None else None
        B, T, H, dk = q.shape
        dv = v.shape[-1]
        o = torch.empty((B, T, H, dv), dtype=q.dtype, device=q.device)
        out = torch.empty((B, H, dk, dv), dtype=torch.float32, device=q.device)
        a = _attention_args(q, k, v, log_decay, lengths, state, scale)
        nbytes = _lib.load().tmpc_decay_attention_workspace_bytes(q.element_size(), ctypes.byref(a), 0)
        ws = _lib.workspace(nbytes, q.device)
        _call(f"tmpc_decay_attention_forward_{sfx}", q.device, ctypes.byref(a), _ptr(o), _ptr(out), _ptr(ws), nbytes)
        if train:
            ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale, ctx.sfx = scale, sfx
        ctx.set_materialize_grads(False)
        return o, out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, d_out):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        dev = q.device
        d_o = _rows(d_o) if d_o is not None else torch.zeros(q.shape[:-1] + v.shape[-1:], dtype=q.dtype, device=dev)
        d_out = d_out.contiguous() if d_out is not None else None
        empty = lambda t: torch.empty(t.shape, dtype=t.dtype, device=dev)  # noqa: E731
        dq, dk, dv = empty(q), empty(k), empty(v)
        d_state = empty(state) if state is not None and ctx.needs_input_grad[4] else None
        a = _attention_args(q, k, v, log_decay, lengths, state, ctx.scale)
        nbytes = _lib.load().tmpc_decay_attention_workspace_bytes(q.element_size(), ctypes.byref(a), 1)
        ws = _lib.workspace(nbytes, dev)
        st = (ctypes.c_int64 * 3)(*d_o.stride()[:3])
        _call(f"tmpc_decay_attention_backward_{ctx.sfx}", dev, ctypes.byref(a), _ptr(d_o), st, _ptr(d_out), _ptr(dq),
              _ptr(dk), _ptr(dv), _ptr(d_state), _ptr(ws), nbytes)
        return dq, dk, dv, None, d_state, None, None, None, None


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                    state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Linear attention with a decay for each head over whole histories.

    q (B, T, H, dk), k (B, T, Hk, dk), v (B, T, Hk, dv), H a multiple of Hk,
    widths 1 to 128; log_decay (H,) float32, <= 0, a constant.  Per problem and head
      S_t = exp(log_decay) S_{t-1} + k_t^T v_t,  o_t = scale q_t S_t,
    from state (B, H, dk, dv) float32 (zero where None), for t < lengths[b]
    (int32, clamped to 0..T; None: T); later steps give zero rows, and what
    their inputs hold is not read.  scale is dk^-1/2 where None.  Returns o
    (B, T, H, dv) and the state after each history's last step (float32)."""
    sfx, scale = _check_attention(q, k, v, log_decay, scale, False)
    B, _, H, dk = q.shape
    if state is not None:
        _check("state", state, q, (B, H, dk, v.shape[-1]), torch.float32)
    if lengths is not None:
        _check("lengths", lengths, q, (B,), torch.int32)
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, state))
    return _DecayAttention.apply(q, k, v, log_decay, state, lengths, scale, sfx, train)


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                         state: torch.Tensor, active: Optional[torch.Tensor] = None,
                         scale: Optional[float] = None) -> torch.Tensor:
    """One step of decay_attention for each problem: q (B, H, dk), k (B, Hk, dk),
    v (B, Hk, dv).  state (B, H, dk, dv), float32 and contiguous, is updated in
    place; returns o (B, H, dv).  Problems whose `active` (B,) bool is False keep
    their state and give zero.  Not differentiable."""
    sfx, scale = _check_attention(q, k, v, log_decay, scale, True)
    B, H, dk = q.shape
    dv = v.shape[-1]
    _check("state", state, q, (B, H, dk, dv), torch.float32)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    if active is not None:
        _check("active", active, q, (B,), torch.bool)
        active = active.contiguous()
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state)):
        raise ValueError("decay_attention_step has no gradient; use decay_attention, or torch.no_grad()")
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    o = torch.empty((B, H, dv), dtype=q.dtype, device=q.device)
    a = _attention_args(q, k, v, log_decay, None, None, scale, step=True)
    _call(f"tmpc_decay_attention_step_{sfx}", q.device, ctypes.byref(a), _ptr(active), _ptr(state), _ptr(o))
    return o


# ---------------------------------------------------------- feed-forward --
class _GatedFF(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act, sfx, train):
        xm = _matrix(x)
        w_gate, w_up, w_down = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
        a = _GatedFF.args(xm, w_gate, w_up, w_down, act)
        M, F = a.M, a.F
        y = torch.empty(x.shape[:-1] + (a.Dout,), dtype=x.dtype, device=x.device)
        gate = torch.empty((M, F), dtype=torch.float32, device=x.device) if train else None
        up = torch.empty((M, F), dtype=torch.float32, device=x.device) if train else None
        nbytes = _lib.load().tmpc_gated_ff_workspace_bytes(x.element_size(), ctypes.byref(a), 0)
        ws = _lib.workspace(nbytes, x.device)
        _call(f"tmpc_gated_ff_forward_{sfx}", x.device, ctypes.byref(a), _ptr(y), _ptr(gate), _ptr(up), _ptr(ws), nbytes)
        if train:
            ctx.save_for_backward(xm, w_gate, w_up, w_down, gate, up)
        ctx.shape, ctx.act, ctx.sfx = x.shape, act, sfx
        return y

    @staticmethod
    def args(xm, w_gate, w_up, w_down, act):
        return _lib.GatedFF(M=xm.shape[0], D=xm.shape[1], F=w_gate.shape[0], Dout=w_down.shape[0], activation=act,
                            x=_ptr(xm), ldx=xm.stride(0), w_gate=_ptr(w_gate), w_up=_ptr(w_up), w_down=_ptr(w_down))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xm, w_gate, w_up, w_down, gate, up = ctx.saved_tensors
        a = _GatedFF.args(xm, w_gate, w_up, w_down, ctx.act)
        dym = _matrix(dy)
        dx = torch.empty(ctx.shape, dtype=xm.dtype, device=xm.device)
        dg, du, dd = torch.empty_like(w_gate), torch.empty_like(w_up), torch.empty_like(w_down)
        nbytes = _lib.load().tmpc_gated_ff_workspace_bytes(xm.element_size(), ctypes.byref(a), 1)
        ws = _lib.workspace(nbytes, xm.device)
        _call(f"tmpc_gated_ff_backward_{ctx.sfx}", xm.device, ctypes.byref(a), _ptr(gate), _ptr(up), _ptr(dym),
              dym.stride(0), _ptr(dx), _ptr(dg), _ptr(du), _ptr(dd), _ptr(ws), nbytes)
        return dx, dg, du, dd, None, None, None


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       activation: str = "silu") -> torch.Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T over the last axis of x (..., D):
    w_gate, w_up (F, D), w_down (Dout, F), activation "silu" or "gelu" (exact)."""
    sfx = _first("x", x, range(1, 9))
    D = x.shape[-1]
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; use one of {', '.join(_ACTIVATIONS)}")
    _check("w_gate", w_gate, x)
    if w_gate.dim() != 2 or w_gate.shape[1] != D or D < 1 or w_gate.shape[0] < 1:
        raise ValueError(f"w_gate has shape {tuple(w_gate.shape)}, expected ('F', {D}), neither empty")
    F = w_gate.shape[0]
    _check("w_up", w_up, x, (F, D))
    _check("w_down", w_down, x)
    if w_down.dim() != 2 or w_down.shape[1] != F or w_down.shape[0] < 1:
        raise ValueError(f"w_down has shape {tuple(w_down.shape)}, expected ('Dout', {F}), not empty")
    train = torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up, w_down))
    return _GatedFF.apply(x, w_gate, w_up, w_down, _ACTIVATIONS[activation], sfx, train)
