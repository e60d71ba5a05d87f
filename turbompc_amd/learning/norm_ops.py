"""Layer norm and dropout with torch autograd, under the rules of `ops`: float32 or
bfloat16 tensors on one HIP device, enqueued on its current stream, statistics in
float32.

Dropout's mask is a function of a key, a call number and an element's place, so it
is made again in the backward pass and never stored.  The key is an int64 tensor
of two on the device, (seed, step): a training loop, or a captured graph of a
step, adds one to key[1] after each step's backward pass (before it, autograd
raises: the backward pass reads the key again) and numbers the calls of a step.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .ops import MAX_NORM_WIDTH, _call, _check, _first, _matrix, _ptr, _wants_grad, _workspace

MAX_DROPOUT_WIDTH = 1 << 24
MAX_DROPOUT_ROWS = (1 << 31) - 1


def _check_dropout(x, p, key, call, what):
    """p as a float; the key's and call's checks where something is dropped."""
    if not (0.0 <= p < 1.0 and round(p * 65536) < 65536):
        raise ValueError(f"{what} must be at least 0 and less than 1 - 2^-17, got {p}")
    if isinstance(call, bool) or not isinstance(call, int) or not 0 <= call < 1 << 32:
        raise ValueError(f"call must be a whole number from 0 to 2^32 - 1, got {call!r}")
    if p == 0.0 and key is None:
        return 0.0
    if key is None:
        raise ValueError(f"{what} {p} needs a key: an int64 tensor (seed, step)")
    _check("key", key, x, (2,), torch.int64)
    if p > 0.0 and x.numel() // x.shape[-1] > MAX_DROPOUT_ROWS:
        raise ValueError(f"x has {x.numel() // x.shape[-1]} rows, expected at most {MAX_DROPOUT_ROWS}")
    return float(p)


# --------------------------------------------------------------- dropout --
def _dropout_run(x, p, key, call, sfx):
    xm, ldx = _matrix(x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    _call(f"tmpc_dropout_{sfx}", x.device, xm.shape[0], xm.shape[1], _ptr(xm), ldx, p, _ptr(key), call, _ptr(y))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, key, call, sfx):
        ctx.save_for_backward(key)
        ctx.args = p, call, sfx
        return _dropout_run(x, p, key, call, sfx)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, call, sfx = ctx.args
        return _dropout_run(dy, p, ctx.saved_tensors[0].contiguous(), call, sfx), None, None, None, None


def dropout(x: torch.Tensor, p: float, key: Optional[torch.Tensor] = None, call: int = 0) -> torch.Tensor:
    """x with each element dropped (set to zero, whatever it holds) with probability p, taken to the
    nearest 2^-16, and the others divided by the share kept.

    The mask follows from key (2,) int64 = (seed, step; its low 32 bits count), `call`
    (0 .. 2^32 - 1: the calls of a step have numbers of their own) and the element's
    place: its row among all rows (the axes before the last, flattened; less than 2^31)
    and its column (rows of 1 to 2^24).  Equal arguments give equal masks, whatever the type and
    strides of x; include/tmpc.h has the generator's definition.  p = 0 returns x."""
    sfx = _first("x", x, range(1, 9))
    D = x.shape[-1]
    if not 1 <= D <= MAX_DROPOUT_WIDTH:
        raise ValueError(f"x has rows of {D} elements, expected 1 to {MAX_DROPOUT_WIDTH}")
    p = _check_dropout(x, p, key, call, "p")
    if p == 0.0:
        return x
    key = key.contiguous()
    if _wants_grad(x):
        return _Dropout.apply(x, p, key, call, sfx)
    return _dropout_run(x, p, key, call, sfx)


# ------------------------------------------------------------------ norm --
_LAYER_NORM = struct.Struct("@qiI4P2q2dP")  # tmpc_layer_norm, packed
assert _LAYER_NORM.size == ctypes.sizeof(_lib.LayerNorm)


def _norm_args(rows, width, call, x, residual, weight, bias, ldx, ldr, eps, p, key):
    at = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
    return _lib.LayerNorm.from_buffer_copy(_LAYER_NORM.pack(rows, width, call, at(x), at(residual), at(weight),
                                                            at(bias), ldx, ldr, eps, p, at(key)))


def _norm_forward(x, residual, weight, bias, eps, p, key, call, sfx, stats):
    """(y, s); stats: a (rows, 2) tensor to fill, or None."""
    xm, ldx = _matrix(x)
    rm, ldr = _matrix(residual) if residual is not None else (None, 0)
    y, s = (torch.empty_like(x, memory_format=torch.contiguous_format) for _ in range(2))
    a = _norm_args(xm.shape[0], xm.shape[1], call, xm, rm, weight, bias, ldx, ldr, eps, p, key)
    _call(f"tmpc_layer_norm_forward_{sfx}", x.device, a, _ptr(y), _ptr(s), _ptr(stats))
    return y, s


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, p, key, call, sfx):
        stats = torch.empty((x.numel() // x.shape[-1], 2), dtype=torch.float32, device=x.device)
        y, s = _norm_forward(x, residual, weight, bias, eps, p, key, call, sfx, stats)
        ctx.args = eps, p, call, sfx, residual is not None, bias is not None
        if x.dtype is torch.bfloat16 and (residual is not None or p > 0.0):  # s was rounded
            saved = None, x, residual
        else:
            saved = s, None, None
        ctx.save_for_backward(*saved, weight, stats, key if p > 0.0 else None)
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds):
        s, x, residual, w, stats, key = ctx.saved_tensors
        eps, p, call, sfx, has_residual, has_bias = ctx.args
        first = s if s is not None else x
        D, dev = first.shape[-1], first.device
        M = first.numel() // D
        matrix = lambda t: _matrix(t) if t is not None else (None, 0)  # noqa: E731
        dym, lddy = _matrix(dy) if dy is not None else (torch.zeros((M, D), dtype=w.dtype, device=dev), D)
        (dsm, ldds), (sm, lds), (xm, ldx), (rm, ldr) = matrix(ds), matrix(s), matrix(x), matrix(residual)
        # a hook may give a tensor back in another layout
        w, stats, key = w.contiguous(), stats.contiguous(), key.contiguous() if key is not None else None
        like = lambda t: torch.empty_like(t, memory_format=torch.contiguous_format)  # noqa: E731
        dx, dw, db = like(first), like(w), like(w) if has_bias else None
        dr = like(first) if has_residual and p > 0.0 else None  # else it is dx
        nbytes, ws = _workspace("tmpc_layer_norm_backward_workspace_bytes", dev, w.element_size(), M, D)
        a = _norm_args(M, D, call, xm, rm, w, None, ldx, ldr, eps, p, key)
        _call(f"tmpc_layer_norm_backward_{sfx}", dev, a, _ptr(dym), lddy, _ptr(dsm), ldds, _ptr(sm), lds,
              _ptr(stats), _ptr(dx), _ptr(dr), _ptr(dw), _ptr(db), _ptr(ws), nbytes)
        return dx, (dx if dr is None else dr) if has_residual else None, dw, db, None, None, None, None, None


def layer_norm_residual(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                        bias: Optional[torch.Tensor] = None, eps: float = 1e-5, dropout: float = 0.0,
                        key: Optional[torch.Tensor] = None, call: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, s): s = d(x) + residual (d(x) where residual is None) and
    y = (s - mean(s)) / sqrt(mean((s - mean(s))^2) + eps) * weight + bias over the last axis (at
    most 8192 wide), d(x) being `dropout(x, dropout, key, call)`.  y is formed from the unrounded
    sum, and so are the gradients."""
    sfx = _first("x", x, range(1, 9))
    D = x.shape[-1]
    if not 1 <= D <= MAX_NORM_WIDTH:
        raise ValueError(f"x has rows of {D} elements, expected 1 to {MAX_NORM_WIDTH}")
    if residual is not None:
        _check("residual", residual, x, x.shape)
    _check("weight", weight, x, (D,))
    if bias is not None:
        _check("bias", bias, x, (D,))
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    p = _check_dropout(x, dropout, key, call, "dropout")
    weight, bias = weight.contiguous(), bias.contiguous() if bias is not None else None
    args = x, residual, weight, bias, float(eps), p, key.contiguous() if p > 0.0 else None, call, sfx
    if _wants_grad(x, residual, weight, bias):
        return _LayerNorm.apply(*args)
    return _norm_forward(*args, None)
