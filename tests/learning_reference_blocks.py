"""Dropout and the layer norm in 64 bits on the CPU, from their definitions, with derived bounds
on a kernel's rounding: each function returns (value, tolerance) for every output."""
import numpy as np
import torch

from learning_reference import F32, cpu64, unit


def philox(counter, key):
    """Philox-4x32-10: four 32-bit words (arrays) of a counter and two of a key."""
    x = [np.asarray(c, dtype=np.uint64) for c in counter]
    shape = np.broadcast_shapes(*(c.shape for c in x))
    x = [np.broadcast_to(c, shape) for c in x]
    low = np.uint64(0xFFFFFFFF)
    for r in range(10):
        k = [np.uint64((key[0] + r * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + r * 0xBB67AE85) % 2 ** 32)]
        a, b = np.uint64(0xD2511F53) * x[0], np.uint64(0xCD9E8D57) * x[2]
        x = [(b >> np.uint64(32)) ^ x[1] ^ k[0], b & low, (a >> np.uint64(32)) ^ x[3] ^ k[1], a & low]
    return x


def kept(M, D, p, key, call):
    """(mask, factor): which elements of (M, D) stay, and what they are multiplied by."""
    seed, step = (int(k) for k in key)
    pieces = (D + 7) // 8
    words = philox((np.arange(pieces)[None], np.arange(M)[:, None], call, step % 2 ** 32),
                   (seed % 2 ** 32, (seed >> 32) % 2 ** 32))
    bits = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=-1)
    least = round(p * 65536)
    mask = torch.from_numpy(bits.reshape(M, 8 * pieces)[:, :D].astype(np.int64)) >= least
    return mask, 65536 / (65536 - least)


def layer_norm(x, r, w, b, eps, dy=None, ds=None, p=0.0, key=None, call=0):
    """{"y", "s"} and, with dy, {"dx", "dr", "dw", "db"}."""
    e = unit(x.dtype)
    x, r, w, b, dy, ds = (cpu64(t) for t in (x, r, w, b, dy, ds))
    M, D = x.shape
    mask, f = kept(M, D, p, key, call) if p > 0 else (torch.ones(M, D, dtype=torch.bool), 1.0)
    drop = lambda t: torch.where(mask, t * f, torch.zeros((), dtype=torch.float64))  # noqa: E731
    parts = drop(x).abs() + (0 if r is None else r.abs())
    s = drop(x) + (0 if r is None else r)
    acc = (D + 32) * 2 * F32  # a sum of D terms
    mean = s.mean(1, keepdim=True)
    c = s - mean
    # the factor, its product and the sum each round once; so do the mean's quotient and the difference
    ec = 4 * F32 * parts + (acc + 4 * F32) * s.abs().mean(1, keepdim=True) + F32 * c.abs()
    var = (c * c).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    evar = (2 * c.abs() * ec + ec * ec).mean(1, keepdim=True) + acc * var
    erel = 0.5 * evar / (var + eps) * (1 + evar / (var + eps)) + 8 * F32  # of rstd
    h = c * rstd
    eh = rstd * ec + h.abs() * (erel + 2 * F32)
    bias = 0 if b is None else b
    y = h * w + bias
    out = {"y": (y, (1 + e) * (eh * w.abs() + 4 * F32 * ((h * w).abs() + abs(bias))) + e * y.abs()),
           "s": (s, 4 * F32 * parts + e * (s.abs() + 4 * F32 * parts))}
    if dy is None:
        return out
    # the backward pass reads the forward pass' statistics, and s as stored where that is in 32 bits
    eh = eh + rstd * (e if e == F32 else 4 * F32) * s.abs()
    a = dy * w
    ma, mah = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
    ema = (acc + 2 * F32) * a.abs().mean(1, keepdim=True)
    emah = (a.abs() * eh).mean(1, keepdim=True) + (acc + 4 * F32) * ((a * h).abs() + a.abs() * eh).mean(1, keepdim=True)
    size = rstd * (a.abs() + ma.abs() + (h * mah).abs())
    dr = rstd * (a - ma - h * mah) + (0 if ds is None else ds)
    edr = rstd * (ema + eh * mah.abs() + (h.abs() + eh) * emah) + size * (erel + 8 * F32) + 2 * F32 * dr.abs()
    out["dr"] = (dr, (1 + e) * edr + e * dr.abs())
    dx = drop(dr)
    out["dx"] = (dx, (1 + e) * (drop(edr) + 2 * F32 * dx.abs()) + e * dx.abs())
    sums = (M + 32) * 2 * F32
    dw, db = (dy * h).sum(0), dy.sum(0)
    edw = (dy.abs() * eh).sum(0) + sums * (dy.abs() * (h.abs() + eh)).sum(0)
    out["dw"] = (dw, (1 + e) * edw + e * dw.abs())
    out["db"] = (db, (1 + e) * sums * dy.abs().sum(0) + e * db.abs())
    return out
