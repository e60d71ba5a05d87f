"""The history model's operators with torch autograd.

Data are float32 or bfloat16 tensors on one HIP device (the parameters of a call
in the same type); states and statistics are float32.  Every call is enqueued on
`torch.cuda.current_stream()` of that device and waits for nothing.  Rows (the
last axis) are read in place when contiguous, whatever the other strides, and
copied otherwise.  Shapes, types and devices that a kernel does not take raise
ValueError or TypeError before anything is enqueued; a failure in the library
raises TmpcError.  There is no CPU path.  Forward-mode derivatives are refused
(NotImplementedError).
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from .. import _lib

_SUFFIX = {torch.float32: "f32", torch.bfloat16: "bf16"}
_ACTIVATIONS = {"silu": 0, "gelu": 1}
MAX_HEAD_WIDTH = 128
MAX_HEADS = 32768
MAX_STEPS = 1 << 30
MAX_BATCH_HEADS = 1 << 23
MAX_NORM_WIDTH = 8192
MAX_FF_WIDTH = 1 << 20
MAX_FF_ROWS = 1 << 30


def _check(name: str, t: torch.Tensor, like: torch.Tensor, shape=None, dtype=None):
    """t has like's device and `dtype` (like's where None) and `shape`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype is not (like.dtype if dtype is None else dtype):
        raise TypeError(f"{name} has dtype {t.dtype}, expected {like.dtype if dtype is None else dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _first(name: str, t: torch.Tensor, dims) -> str:
    """The suffix of the call whose first argument is t."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    sfx = _SUFFIX.get(t.dtype)
    if sfx is None:
        raise TypeError(f"unsupported dtype {t.dtype}; use float32 or bfloat16")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}; the operators run on a HIP device")
    if t.dim() not in dims:
        raise ValueError(f"{name} has {t.dim()} dimensions, expected {' or '.join(map(str, dims))}")
    return sfx


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous rows: itself where it has them."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


# An axis of one entry may have any stride, which a copy keeps: the calls get one of their own.
def _steps(t: torch.Tensor) -> torch.Tensor:
    """A history (B, T, H, d) as the kernels read it: contiguous rows, steps less than 2^23
    elements apart."""
    return t if (t.stride(-1) == 1 or t.shape[-1] <= 1) and _step_strides(t)[1] < 1 << 23 else t.contiguous()


def _step_strides(t: torch.Tensor) -> Tuple[int, int, int]:
    """Strides of problem, step and head of a history (B, T, H, d), or of one step of each (B, H, d)."""
    s = t.stride()
    if t.dim() == 3:
        return s[0], 0, s[1]
    return s[0], s[1] if t.shape[1] > 1 else 0, s[2]


def _matrix(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """t as (rows, last axis) with contiguous rows, at most 2^20 elements apart (a view where one
    exists), and the elements between its rows."""
    t = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    rows, width = t.shape
    pitch = t.stride(0) if rows > 1 else width
    if (width <= 1 or t.stride(1) == 1) and pitch <= MAX_FF_WIDTH:
        return t, pitch
    return t.contiguous(), width


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return (t.data_ptr() or None) if t is not None else None  # an empty tensor's is null


def _wants_grad(*ts: Optional[torch.Tensor]) -> bool:
    # a tangent is no matter of requires_grad or grad mode; outside a level there are none
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the history model's operators have no forward-mode derivatives")
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


_FUNCTIONS = {}


def _call(fn: str, device: torch.device, *args):
    f = _FUNCTIONS.get(fn)
    if f is None:
        f = _FUNCTIONS[fn] = getattr(_lib.load(), fn)
    if device.index == torch.cuda.current_device():
        _lib.check(fn, f(torch._C._cuda_getCurrentRawStream(device.index), *args))
    else:
        with torch.cuda.device(device):
            _lib.check(fn, f(_lib.stream_handle(device), *args))


def _workspace(query: str, device: torch.device, *args):
    """(bytes, tensor or None) of a call's workspace."""
    nbytes = getattr(_lib.load(), query)(*args)
    return nbytes, torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


# ------------------------------------------------------------------ norm --
def _rms_forward(x, residual, weight, eps, sfx, rstd):
    """(y, s); rstd: a (rows,) tensor to fill, or None."""
    xm, ldx = _matrix(x)
    rm, ldr = _matrix(residual) if residual is not None else (None, 0)
    M, D = xm.shape
    y, s = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for _ in range(2))
    _call(f"tmpc_rms_norm_forward_{sfx}", x.device, M, D, _ptr(xm), ldx, _ptr(rm), ldr,
          _ptr(weight), eps, _ptr(y), _ptr(s), _ptr(rstd))
    return y, s


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, sfx):
        rstd = torch.empty(x.numel() // x.shape[-1], dtype=torch.float32, device=x.device)
        y, s = _rms_forward(x, residual, weight, eps, sfx, rstd)
        ctx.sfx, ctx.has_residual = sfx, residual is not None
        ctx.save_for_backward(s, weight, rstd)
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds):
        s, w, rstd = ctx.saved_tensors
        D = s.shape[-1]
        M = s.numel() // D
        dym, lddy = _matrix(dy) if dy is not None else (torch.zeros((M, D), dtype=s.dtype, device=s.device), D)
        dsm, ldds = _matrix(ds) if ds is not None else (None, 0)
        dx, dw = torch.empty_like(s), torch.empty_like(w)
        nbytes, ws = _workspace("tmpc_rms_norm_backward_workspace_bytes", s.device, s.element_size(), M, D)
        _call(f"tmpc_rms_norm_backward_{ctx.sfx}", s.device, M, D, _ptr(dym), lddy, _ptr(dsm), ldds,
              _ptr(s), D, _ptr(w), _ptr(rstd), _ptr(dx), _ptr(dw), _ptr(ws), nbytes)
        return dx, dx if ctx.has_residual else None, dw, None, None


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
    weight, eps = weight.contiguous(), float(eps)
    if _wants_grad(x, residual, weight):
        return _RmsNorm.apply(x, residual, weight, eps, sfx)
    return _rms_forward(x, residual, weight, eps, sfx, None)


# ------------------------------------------------------------- attention --
# tmpc_decay_attention, packed (its fields are naturally aligned)
_ATTENTION = struct.Struct("@6i3P9q3Pd")
assert _ATTENTION.size == ctypes.sizeof(_lib.DecayAttention)


def _attention_args(q, k, v, log_decay, lengths, state, scale):
    B, T, H, dk = q.shape if q.dim() == 4 else (q.shape[0], 1) + q.shape[1:]
    p = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
    return _lib.DecayAttention.from_buffer_copy(_ATTENTION.pack(
        B, T, H, k.shape[-2], dk, v.shape[-1], p(q), p(k), p(v), *_step_strides(q), *_step_strides(k),
        *_step_strides(v), p(log_decay), p(lengths), p(state), scale))


def _check_attention(q, k, v, log_decay, scale, step):
    sfx = _first("q", q, (3,) if step else (4,))
    _check("k", k, q)
    _check("v", v, q)
    qs, ks, vs = q.shape, k.shape, v.shape
    lead, (H, dk) = qs[:-2], qs[-2:]
    if len(ks) != len(qs) or ks[:-2] != lead or ks[-1] != dk:
        raise ValueError(f"k has shape {tuple(ks)}, expected {tuple(lead) + ('Hk', dk)}")
    Hk = ks[-2]
    if len(vs) != len(qs) or vs[:-1] != ks[:-1]:
        raise ValueError(f"v has shape {tuple(vs)}, expected {tuple(lead) + (Hk, 'dv')}")
    if H < 1 or Hk < 1 or H % Hk:
        raise ValueError(f"the {H} heads of q are not a multiple of the {Hk} heads of k and v")
    if H > MAX_HEADS:
        raise ValueError(f"q has {H} heads, expected at most {MAX_HEADS}")
    if qs[0] * H > MAX_BATCH_HEADS:
        raise ValueError(f"q has {qs[0]} problems of {H} heads, expected at most {MAX_BATCH_HEADS} together")
    if not step and qs[1] > MAX_STEPS:
        raise ValueError(f"q has {qs[1]} steps, expected at most {MAX_STEPS}")
    for name, d in (("q and k", dk), ("v", vs[-1])):
        if not 1 <= d <= MAX_HEAD_WIDTH:
            raise ValueError(f"{name} have heads of {d} elements, expected 1 to {MAX_HEAD_WIDTH}")
    _check("log_decay", log_decay, q, (H,), torch.float32)
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant of the model: it takes no gradient")
    return sfx, float(dk ** -0.5 if scale is None else scale)


def _attention_forward(q, k, v, log_decay, state, lengths, scale, sfx):
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    o = torch.empty((B, T, H, dv), dtype=q.dtype, device=q.device)
    out = torch.empty((B, H, dk, dv), dtype=torch.float32, device=q.device)
    a = _attention_args(q, k, v, log_decay, lengths, state, scale)
    nbytes, ws = _workspace("tmpc_decay_attention_workspace_bytes", q.device, q.element_size(), a, 0)
    _call(f"tmpc_decay_attention_forward_{sfx}", q.device, a, _ptr(o), _ptr(out), _ptr(ws), nbytes)
    return o, out


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale, sfx):
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale, ctx.sfx = scale, sfx
        ctx.set_materialize_grads(False)
        return _attention_forward(q, k, v, log_decay, state, lengths, scale, sfx)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, d_out):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        dev = q.device
        d_o = _steps(d_o) if d_o is not None else torch.zeros(q.shape[:-1] + v.shape[-1:], dtype=q.dtype, device=dev)
        d_out = d_out.contiguous() if d_out is not None else None
        empty = lambda t: torch.empty(t.shape, dtype=t.dtype, device=dev)  # noqa: E731
        dq, dk, dv = empty(q), empty(k), empty(v)
        d_state = empty(state) if state is not None and ctx.needs_input_grad[4] else None
        a = _attention_args(q, k, v, log_decay, lengths, state, ctx.scale)
        nbytes, ws = _workspace("tmpc_decay_attention_workspace_bytes", dev, q.element_size(), a, 1)
        st = (ctypes.c_int64 * 3)(*_step_strides(d_o))
        _call(f"tmpc_decay_attention_backward_{ctx.sfx}", dev, a, _ptr(d_o), st, _ptr(d_out), _ptr(dq), _ptr(dk),
              _ptr(dv), _ptr(d_state), _ptr(ws), nbytes)
        return dq, dk, dv, None, d_state, None, None, None


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                    state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Linear attention with a decay for each head over whole histories.

    q (B, T, H, dk), k (B, T, Hk, dk), v (B, T, Hk, dv), H a multiple of Hk,
    T at most 2^30, widths 1 to 128; log_decay (H,) float32, <= 0, a constant.  Per problem and head
      S_t = exp(log_decay) S_{t-1} + k_t^T v_t,  o_t = scale q_t S_t,
    from state (B, H, dk, dv) float32 (zero where None), for t < lengths[b]
    (int32, clamped to 0..T; None: T); later steps give zero rows, and what
    their inputs hold is not read.  An infinite or NaN value at a live step spoils
    what it has a part in: no earlier step, other head or problem.  scale is dk^-1/2 where None.  Returns o
    (B, T, H, dv) and the state after each history's last step (float32)."""
    sfx, scale = _check_attention(q, k, v, log_decay, scale, False)
    B, _, H, dk = q.shape
    if state is not None:
        _check("state", state, q, (B, H, dk, v.shape[-1]), torch.float32)
    if lengths is not None:
        _check("lengths", lengths, q, (B,), torch.int32)
    state = state.contiguous() if state is not None else None
    lengths = lengths.contiguous() if lengths is not None else None
    args = (_steps(q), _steps(k), _steps(v), log_decay.contiguous(), state, lengths, scale, sfx)
    return _DecayAttention.apply(*args) if _wants_grad(q, k, v, state, log_decay) else _attention_forward(*args)


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
    if _wants_grad(q, k, v, state, log_decay):
        raise ValueError("decay_attention_step has no gradient; use decay_attention, or torch.no_grad()")
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    o = torch.empty((B, H, dv), dtype=q.dtype, device=q.device)
    a = _attention_args(q, k, v, log_decay, None, None, scale)
    _call(f"tmpc_decay_attention_step_{sfx}", q.device, a, _ptr(active), _ptr(state), _ptr(o))
    increment_version(state)  # a backward pass that saved it has to see the change
    return o


# ---------------------------------------------------------- feed-forward --
_GATED_FF = struct.Struct("@q4iPq3P")  # tmpc_gated_ff, packed
assert _GATED_FF.size == ctypes.sizeof(_lib.GatedFF)


def _ff_args(xm, ldx, w_gate, w_up, w_down, act):
    F, D = w_gate.shape
    return _lib.GatedFF.from_buffer_copy(_GATED_FF.pack(xm.shape[0], D, F, w_down.shape[0], act, xm.data_ptr(),
                                                        ldx, w_gate.data_ptr(), w_up.data_ptr(),
                                                        w_down.data_ptr()))


def _ff_forward(x, xm, ldx, w_gate, w_up, w_down, act, sfx, gate, up):
    """y; gate, up: fp32 tensors to fill, or None."""
    a = _ff_args(xm, ldx, w_gate, w_up, w_down, act)
    y = torch.empty(x.shape[:-1] + (w_down.shape[0],), dtype=x.dtype, device=x.device)
    nbytes, ws = _workspace("tmpc_gated_ff_workspace_bytes", x.device, x.element_size(), a, 0)
    _call(f"tmpc_gated_ff_forward_{sfx}", x.device, a, _ptr(y), _ptr(gate), _ptr(up), _ptr(ws), nbytes)
    return y


class _GatedFF(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act, sfx):
        xm, ldx = _matrix(x)
        gate, up = (torch.empty((xm.shape[0], w_gate.shape[0]), dtype=torch.float32, device=x.device) for _ in range(2))
        ctx.save_for_backward(xm, w_gate, w_up, w_down, gate, up)
        ctx.shape, ctx.act, ctx.sfx = x.shape, act, sfx
        return _ff_forward(x, xm, ldx, w_gate, w_up, w_down, act, sfx, gate, up)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xm, w_gate, w_up, w_down, gate, up = ctx.saved_tensors
        xm, ldx = _matrix(xm)
        a = _ff_args(xm, ldx, w_gate, w_up, w_down, ctx.act)
        dym, lddy = _matrix(dy)
        dx = torch.empty(ctx.shape, dtype=xm.dtype, device=xm.device)
        dg, du, dd = torch.empty_like(w_gate), torch.empty_like(w_up), torch.empty_like(w_down)
        nbytes, ws = _workspace("tmpc_gated_ff_workspace_bytes", xm.device, xm.element_size(), a, 1)
        _call(f"tmpc_gated_ff_backward_{ctx.sfx}", xm.device, a, _ptr(gate), _ptr(up), _ptr(dym),
              lddy, _ptr(dx), _ptr(dg), _ptr(du), _ptr(dd), _ptr(ws), nbytes)
        return dx, dg, du, dd, None, None


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
    if max(D, F, w_down.shape[0]) > MAX_FF_WIDTH:
        raise ValueError(f"the widths of x, w_gate and w_down must be at most {MAX_FF_WIDTH}")
    if x.numel() // D > MAX_FF_ROWS:
        raise ValueError(f"x has {x.numel() // D} rows, expected at most {MAX_FF_ROWS}")
    act = _ACTIVATIONS[activation]
    w_gate, w_up, w_down = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
    if _wants_grad(x, w_gate, w_up, w_down):
        return _GatedFF.apply(x, w_gate, w_up, w_down, act, sfx)
    return _ff_forward(x, *_matrix(x), w_gate, w_up, w_down, act, sfx, None, None)
