"""The gated delta rule in 64 bits on the CPU, step by step from its definition, its derivatives
written out, with bounds on a kernel's rounding.

`delta` returns {name: (value, tolerance, limit)}.  They count two things.

Roundings to the data's type (unit e, 2^-8 for bf16): half a unit of each result, and of operands of
products whose result is of that type.  An output is a product of q with the state at the start of its
block of 16 steps and of scores with the block's u, whose inexact operands keep 16 bits (two terms of 8,
cut off: 2^-15 each, two a product at most); a
gradient of q or k has up to three roundings a product (u, the score, a state), with the states at the
ends of its chunk of 64 steps.  Each is e times the sum of the products' magnitudes; beta's
gradient reads e_t by two rounded terms.  These are elementwise tolerances, zero in fp32.

Roundings in fp32: a step's map of the state, a (I - beta k^T k), lengthens nothing where beta |k|^2
is from 0 to 2, so that errors made at one step are carried on and not raised, and add up as
independent ones: n of them to sqrt(n) units of the norm of a head's values.  With n = T + dk + dv + 64 (the
steps, the sums of a product's terms, a block's inverse and its product) and `chain` products in a
row, chain sqrt(n) units; eight times that is the limit, in the norm of each head, on what the
tolerances leave over.
"""
import torch

from learning_reference import F32, TINY, cpu64, unit

BLOCK, CHUNK = 16, 64


def _loop(q, k, v, g, beta, state, n, scale, do, dstate):
    """The recurrence and its derivatives, all (B, T, H, ...) with heads repeated."""
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    zero = lambda *s: torch.zeros((B, T, H) + s, dtype=torch.float64)  # noqa: E731
    out = {"o": zero(dv), "e": zero(dv), "before": zero(dk, dv)}
    S = torch.zeros((B, H, dk, dv), dtype=torch.float64) if state is None else state.clone()
    a = torch.exp(g)
    for t in range(T):
        on = (t < n)[:, None, None]
        at = a[:, t, :, None]
        out["before"][:, t] = S
        e = v[:, t] - at * (k[:, t, :, None] @ S)[:, :, 0]
        new = at[..., None] * S + k[:, t, :, :, None] * (beta[:, t, :, None] * e)[:, :, None]
        out["o"][:, t] = torch.where(on, scale * (q[:, t, :, None] @ new)[:, :, 0], 0.0)
        out["e"][:, t] = torch.where(on, e, 0.0)
        S = torch.where(on[..., None], new, S)
    out["state"] = S
    if do is None:
        return out
    out.update(dq=zero(dk), dk=zero(dk), y=zero(dv), du=zero(dv), dbeta=zero(), dg=zero(), after=zero(dk, dv))
    R = torch.zeros_like(S) if dstate is None else dstate.clone()

    def put(key, t, on, x):
        out[key][:, t] = torch.where(on if x.dim() == 3 else on[..., 0], x, 0.0)

    for t in range(T - 1, -1, -1):
        on = (t < n)[:, None, None]
        at, S0, e = a[:, t, :, None], out["before"][:, t], out["e"][:, t]
        u = beta[:, t, :, None] * e
        S1 = at[..., None] * S0 + k[:, t, :, :, None] * u[:, :, None]
        out["after"][:, t] = R
        D = R + scale * q[:, t, :, :, None] * do[:, t, :, None]
        du = (k[:, t, :, None] @ D)[:, :, 0]
        y = beta[:, t, :, None] * du
        new = at[..., None] * (D - k[:, t, :, :, None] * y[:, :, None])
        put("dq", t, on, scale * (S1 @ do[:, t, :, :, None])[..., 0])
        put("dk", t, on, (D @ u[..., None])[..., 0] - at * (S0 @ y[..., None])[..., 0])
        put("y", t, on, y)
        put("du", t, on, du)
        put("dbeta", t, on, (du * e).sum(-1))
        put("dg", t, on, (new * S0).sum((-1, -2)))
        R = torch.where(on[..., None], new, R)
    out["dstate"] = R
    return out


def _magnitudes(x, q, k, g, beta, scale, do):
    """The products' magnitudes summed: of o (by blocks), dq and dk (by chunks)."""
    T = q.shape[1]
    u = beta[..., None] * x["e"]
    rows = lambda z, s: z[:, s].transpose(1, 2).abs()  # noqa: E731  (B, H, C, d)

    def spans(size):
        for t0 in range(0, T, size):
            s = slice(t0, min(t0 + size, T))
            G = g[:, s].clamp(min=-1e5).transpose(1, 2).cumsum(-1)
            i = torch.arange(G.shape[-1])
            ratio = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(i[:, None] < i, -float("inf")))
            yield s, torch.exp(G)[..., None], torch.exp(G[..., -1:] - G)[..., None], ratio

    mo, mq, mk = torch.zeros_like(x["o"]), torch.zeros_like(q), torch.zeros_like(k)
    for s, start, _, ratio in spans(BLOCK):
        scores = rows(q, s) @ rows(k, s).transpose(-1, -2) * ratio
        mo[:, s] = abs(scale) * (start * (rows(q, s) @ x["before"][:, s.start].abs()) + scores @ rows(u, s)).transpose(1, 2)
    if do is None:
        return mo, None, None
    for s, start, end, ratio in spans(CHUNK):
        S0, R1 = x["before"][:, s.start].abs().transpose(-1, -2), x["after"][:, s.stop - 1].abs().transpose(-1, -2)
        d, y, w, kk = (rows(z, s) for z in (do, x["y"], u, k))
        m1, m2 = (abs(scale) * d @ w.transpose(-1, -2)) * ratio, (y @ w.transpose(-1, -2)) * ratio
        mq[:, s] = (start * abs(scale) * (d @ S0) + m1 @ kk).transpose(1, 2)
        mk[:, s] = (end * (w @ R1) + start * (y @ S0) + m1.transpose(-1, -2) @ rows(q, s) + m2.transpose(-1, -2) @ kk
                    + m2 @ kk).transpose(1, 2)
    return mo, mq, mk


def norm_limit(T, dk, dv, chain):
    return 8 * chain * (T + dk + dv + 64) ** 0.5 * F32


def delta(q, k, v, g, beta, state=None, lengths=None, scale=None, do=None, dstate=None):
    """{name: (value, elementwise tolerance, limit, other terms of the norm or None)}: "o", "state" and,
    with do, "dq", "dk", "dv", "dg", "dbeta", "dstate"."""
    r = unit(q.dtype) if q.dtype != torch.float32 else 0.0
    B, T, H = g.shape
    heads = {"dq": q.shape[2], "dk": k.shape[2], "dv": v.shape[2]}
    n = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    live = (torch.arange(T) < n[:, None])[..., None]
    f = [cpu64(z).repeat_interleave(H // z.shape[2], 2) for z in (q, k, v)]
    f = [torch.where(live[..., None], z, 0.0) for z in f]
    g, beta = torch.where(live, cpu64(g), 0.0), torch.where(live, cpu64(beta), 0.0)
    do = torch.where(live[..., None], cpu64(do), 0.0) if do is not None else None
    x = _loop(*f, g, beta, cpu64(state), n, scale, do, cpu64(dstate))
    mo, mq, mk = _magnitudes(x, f[0], f[1], g, beta, scale, do)
    dk, dv = q.shape[-1], v.shape[-1]
    lim = lambda c: norm_limit(T, dk, dv, c)  # noqa: E731
    # 1.02: what is of second order, and the exponentials' own error
    out = {"o": (x["o"], r * x["o"].abs() + 1.02 * 4 * r * r * mo, lim(3), None), "state": (x["state"], 0.0, lim(3), None)}
    if do is None:
        return out
    group = lambda z, key: z.reshape(B, T, heads[key], H // heads[key], -1).sum(3)  # noqa: E731
    for key, val, mag in (("dq", x["dq"], mq), ("dk", x["dk"], mk)):
        total = group(val, key)
        out[key] = (total, r * total.abs() + 1.02 * 3 * r * group(mag, key), lim(6), None)
    total = group(x["y"], "dv")
    out["dv"] = (total, r * total.abs(), lim(5), None)
    out["dbeta"] = (x["dbeta"], r * x["dbeta"].abs() + 1.02 * r * r * (x["du"].abs() * x["e"].abs()).sum(-1), lim(6), None)
    # log_decay's gradient is summed up from terms do . o - dv . v: its errors are units of those too
    terms = torch.stack([(do.abs() * x["o"].abs()).sum(-1), (x["y"].abs() * f[2].abs()).sum(-1)], -1)
    out["dg"] = (x["dg"], 0.0, lim(6), terms)
    out["dstate"] = (x["dstate"], 0.0, lim(5), None)
    return out


def assert_within(name, got, want, head_axis):
    """What is left of got's error above the tolerance is within the limit, head by head."""
    value, tol, limit, terms = want
    got = cpu64(got)
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert bool(torch.isfinite(got).all()), name
    if not got.numel():
        return
    norm = lambda z: z.movedim((0, head_axis), (0, 1)).flatten(2).norm(dim=-1)  # noqa: E731  (B, heads)
    over = norm(((got - value).abs() - tol).clamp(min=0))
    most = limit * (norm(value) + (norm(terms) if terms is not None else 0.0)) + TINY
    worst = float((over / most).max())
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound at problem and head {divmod(int((over / most).argmax()), over.shape[1])}"
