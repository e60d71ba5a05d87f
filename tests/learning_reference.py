"""The history model's operators in 64 bits on the CPU, step by step from their
definitions, with derived bounds on a kernel's rounding.

Each function returns, for every output, (value, magnitude): the magnitude is the
same formula on absolute values, so an evaluation whose every product and partial
sum is rounded with relative error eps differs by at most about (number of
roundings) * eps * magnitude, whatever cancels.
"""
import math

import torch

F32 = 2.0 ** -24  # unit roundoffs
BF16 = 2.0 ** -8  # 8 significand bits
TINY = 2.0 ** -120  # sums of values that underflow in fp32 (below 2^-126)


def unit(dtype):
    return F32 if dtype == torch.float32 else BF16


def cpu64(t):
    return t.detach().cpu().double() if t is not None else None


def attention(q, k, v, g, state=None, lengths=None, scale=None, do=None, dstate=None):
    """{"o", "state"} and, with do, {"dq", "dk", "dv", "dstate"}, each (value, magnitude)."""
    a = [cpu64(t) for t in (q, k, v, state, do, dstate)]
    n = lengths.cpu().long() if lengths is not None else None
    val = _attention(*a, cpu64(g), n, scale)
    mag = _attention(*[t.abs() if t is not None else None for t in a], cpu64(g), n,
                     None if scale is None else abs(scale))
    return {key: (val[key], mag[key]) for key in val}


def _attention(q, k, v, state, do, dstate, g, n, scale):
    B, T, H, dk = q.shape
    Hk, dv = k.shape[2], v.shape[3]
    G = H // Hk
    scale = dk ** -0.5 if scale is None else scale
    gamma = torch.exp(g)[:, None, None]
    n = torch.full((B,), T) if n is None else n.clamp(0, T)
    S = torch.zeros((B, H, dk, dv), dtype=torch.float64) if state is None else state.clone()
    o, dq = torch.zeros((B, T, H, dv), dtype=torch.float64), torch.zeros_like(q)
    gk, gv = torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        for t in range(int(n[b])):
            kt, vt = (x[b, t].repeat_interleave(G, 0) for x in (k, v))
            S[b] = gamma * S[b] + kt[:, :, None] * vt[:, None, :]
            o[b, t] = scale * (q[b, t][:, None, :] @ S[b])[:, 0]
            if do is not None:
                dq[b, t] = scale * (S[b] @ do[b, t][:, :, None])[:, :, 0]
    out = {"o": o, "state": S}
    if do is None:
        return out
    R = torch.zeros_like(S) if dstate is None else dstate.clone()
    for b in range(B):
        for t in range(int(n[b]) - 1, -1, -1):
            R[b] = R[b] + scale * q[b, t][:, :, None] * do[b, t][:, None, :]
            kt, vt = (x[b, t].repeat_interleave(G, 0) for x in (k, v))
            gk[b, t] = (R[b] @ vt[:, :, None])[:, :, 0].reshape(Hk, G, dk).sum(1)
            gv[b, t] = (kt[:, None, :] @ R[b])[:, 0].reshape(Hk, G, dv).sum(1)
            R[b] = gamma * R[b]
    out.update(dq=dq, dk=gk, dv=gv, dstate=R)
    return out


def act(name, g):
    """(act, act', a bound on |act''|)"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), 0.5
    phi = 0.5 * torch.special.erfc(-g / math.sqrt(2))
    pdf = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return g * phi, phi + g * pdf, 0.8


def feed_forward(x, wg, wu, wd, name, dy=None):
    """{"y"} and, with dy, {"dx", "dwg", "dwu", "dwd"}, each (value, tolerance) for data of x's type."""
    e = unit(x.dtype)
    acc = lambda n: (n + 16) * 2 * F32  # noqa: E731  a sum of n products, fp32
    x, wg, wu, wd, dy = (cpu64(t) for t in (x, wg, wu, wd, dy))
    D, F = x.shape[1], wg.shape[0]
    g, u = x @ wg.T, x @ wu.T
    eg, eu = acc(D) * (x.abs() @ wg.abs().T), acc(D) * (x.abs() @ wu.abs().T)
    a, da, dd = act(name, g)
    ea = 1.2 * eg + 8 * F32 * (a.abs() + g.abs())  # |act'| <= 1.13, and the function's own rounding
    h = a * u
    eh = ea * u.abs() + a.abs() * eu + 2 * F32 * h.abs()
    hr = eh + e * h.abs()  # h as an operand
    y = h @ wd.T
    out = {"y": (y, hr @ wd.abs().T + acc(F) * (h.abs() @ wd.abs().T) + e * y.abs())}
    if dy is None:
        return out
    dh = dy @ wd
    edh = acc(dy.shape[1]) * (dy.abs() @ wd.abs())
    eda = dd * eg + 16 * F32 * (1 + g.abs())
    dg, du = dh * u * da, dh * a
    edg = edh * (u * da).abs() + dh.abs() * (eu * da.abs() + u.abs() * eda) + e * dg.abs()
    edu = edh * a.abs() + dh.abs() * ea + e * du.abs()
    M = x.shape[0]
    dx = dg @ wg + du @ wu
    out["dx"] = (dx, edg @ wg.abs() + edu @ wu.abs() + acc(2 * F) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
                 + e * dx.abs())
    for key, p, ep, r in (("dwg", dg, edg, x), ("dwu", du, edu, x), ("dwd", dy, 0 * dy, h)):
        val = p.T @ r
        tol = ep.T @ r.abs() + acc(M) * (p.abs().T @ r.abs()) + e * val.abs()
        if key == "dwd":
            tol = tol + p.abs().T @ hr
        out[key] = (val, tol)
    return out


def norm(x, r, w, eps, dy=None, ds=None):
    """{"y", "s"} and, with dy, {"dx", "dw"}, each (value, tolerance)."""
    e = unit(x.dtype)
    x, r, w, dy, ds = (cpu64(t) for t in (x, r, w, dy, ds))
    D = x.shape[1]
    s = x if r is None else x + r
    rstd = ((s * s).mean(1, keepdim=True) + eps) ** -0.5
    y = s * rstd * w
    acc = (D + 32) * 2 * F32
    out = {"y": (y, (e + acc) * y.abs() + 4 * F32 * (x.abs() + (0 if r is None else r.abs())) * rstd * w.abs()),
           "s": (s, 2 * e * s.abs() + 2 * F32 * (x.abs() + (0 if r is None else r.abs())))}
    if dy is None:
        return out
    a = dy * w
    xh = s * rstd
    m = (a * xh).mean(1, keepdim=True)
    dx = rstd * (a - xh * m) + (0 if ds is None else ds)
    # the backward pass reads s as stored: each xh off by e, its mean with it
    exh = (e + acc) * xh.abs()
    em = (e + acc) * (a * xh).abs().mean(1, keepdim=True)
    out["dx"] = (dx, rstd * (exh * m.abs() + xh.abs() * em + acc * (a.abs() + (xh * m).abs()))
                 + (e + 4 * F32) * (dx.abs() + (0 if ds is None else ds.abs())))
    dw = (dy * xh).sum(0)
    out["dw"] = (dw, (dy.abs() * exh).sum(0) + (x.shape[0] + 32) * 2 * F32 * (dy * xh).abs().sum(0) + e * dw.abs())
    return out


def assert_within(name, got, value, tol):
    got = cpu64(got)
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert bool(torch.isfinite(got).all()), name
    over = (got - value).abs() - (tol + TINY)
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0.0, f"{name}: {worst:.3e} over its bound at {torch.nonzero(over == over.max())[0].tolist()}"
