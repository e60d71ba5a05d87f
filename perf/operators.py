"""The operators of the history model in front of the differentiable solve: what is measured.

A case is a dict of plain values: `op` and its sizes.  `prepare` makes the
inputs a training or control program holds before the call, `run` makes one
pass through the operator (its plain form in elementary torch operations in 32
bits, or the package's operators where `own` is true), `exact` computes the
same from the definition in 64 bits, and `work` says what a pass cannot do
without.

  step   one control period: single-token decay attention, state updated in place
  attn   decay attention over whole histories; `train` adds its backward pass
  ff     gated feed-forward block; `train` adds its backward pass
  norm   root-mean-square norm of x + residual; `train` adds its backward pass
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
EPS = 1e-6
PLAIN_CHUNK = 128


def listed():
    return [
        # 64 vehicles (the point-mass batch), one control period of a small model: latency
        {"name": "step_64_f32", "op": "step", "dtype": "f32", "B": 64, "H": 4, "Hk": 4, "dk": 32, "dv": 32,
         "masked": False},
        # the quadrotor batch, one control period, shared key/value heads, some vehicles idle
        {"name": "step_fleet_bf16", "op": "step", "dtype": "bf16", "B": 4096, "H": 8, "Hk": 2, "dk": 64, "dv": 64,
         "masked": True},
        # histories of the LTI suite (1024 problems, 51 stages), ragged, odd head widths, fp32
        {"name": "attn_ragged_f32", "op": "attn", "dtype": "f32", "B": 1024, "T": 51, "H": 4, "Hk": 2, "dk": 33,
         "dv": 57, "ragged": True, "state": False, "train": False},
        # one very long log of a single vehicle (odd length): few rows, a long axis
        {"name": "attn_long_bf16", "op": "attn", "dtype": "bf16", "B": 1, "T": 50001, "H": 16, "Hk": 16, "dk": 128,
         "dv": 128, "ragged": False, "state": True, "train": False},
        # a training batch of long windows that continue from earlier windows' states
        {"name": "attn_train_bf16", "op": "attn", "dtype": "bf16", "B": 64, "T": 1024, "H": 8, "Hk": 8, "dk": 64,
         "dv": 64, "ragged": False, "state": True, "train": True},
        # the spacecraft batch (2048 problems, 101 stages), ragged, one key/value head for all
        {"name": "attn_train_shared_bf16", "op": "attn", "dtype": "bf16", "B": 2048, "T": 101, "H": 4, "Hk": 1,
         "dk": 64, "dv": 128, "ragged": True, "state": False, "train": True},
        # one control period's rows through a small block: latency
        {"name": "ff_64_bf16", "op": "ff", "dtype": "bf16", "M": 64, "D": 256, "F": 683, "act": "silu",
         "train": False},
        # the largest block: a batch of histories through a wide model
        {"name": "ff_large_bf16", "op": "ff", "dtype": "bf16", "M": 16384, "D": 2048, "F": 5504, "act": "silu",
         "train": False},
        # a training step over 205 histories of 101 stages
        {"name": "ff_train_bf16", "op": "ff", "dtype": "bf16", "M": 20705, "D": 512, "F": 1408, "act": "silu",
         "train": True},
        # the same in fp32 on a small model: 51 histories of 41 stages
        {"name": "ff_train_f32", "op": "ff", "dtype": "f32", "M": 2091, "D": 200, "F": 520, "act": "gelu",
         "train": True},
        # one control period's rows: latency
        {"name": "norm_64_bf16", "op": "norm", "dtype": "bf16", "M": 64, "D": 256, "train": False},
        # every step of the spacecraft batch's histories, training
        {"name": "norm_train_bf16", "op": "norm", "dtype": "bf16", "M": 206848, "D": 512, "train": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "attn", "attn", "ff", "ff", "norm"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    if op in ("step", "attn"):
        Hk = rng.choice([1, 2, 3, 4, 8])
        H = Hk * rng.choice([1, 1, 2, 4])
        dk, dv = (rng.choice([16, 32, 33, 48, 57, 64, 80, 96, 127, 128]) for _ in range(2))
        if op == "step":
            most = 4096 * 8 * 64 * 64 // (H * dk * dv)
            return {"op": op, "dtype": dtype, "B": _log_int(rng, 1, max(1, min(4096, most))), "H": H, "Hk": Hk,
                    "dk": dk, "dv": dv, "masked": rng.random() < 0.5}
        train = rng.random() < 0.5
        T = _log_int(rng, 1, 50001)
        # tokens x heads x widths of the largest listed case of this kind (half of it in fp32)
        most = (2048 * 101 * 4 * 192 if train else 50001 * 16 * 256) * 2 // (BYTES[dtype] * H * (dk + dv))
        T = min(T, most)
        return {"op": op, "dtype": dtype, "B": _log_int(rng, 1, max(1, min(2048, most // T))), "T": T, "H": H,
                "Hk": Hk, "dk": dk, "dv": dv, "ragged": rng.random() < 0.5, "state": rng.random() < 0.5,
                "train": train}
    if op == "ff":
        train = rng.random() < 0.5
        D, F = _log_int(rng, 32, 2048), _log_int(rng, 64, 5504)
        if rng.random() < 0.5:  # half of the models have widths of whole 32-byte pieces
            D, F = (D + 15) // 16 * 16, (F + 15) // 16 * 16
        most = (20705 * 512 * 1408 * 4 if train else 16384 * 2048 * 5504) // (D * F)
        if dtype == "f32":
            most //= 8
        return {"op": op, "dtype": dtype, "M": _log_int(rng, 1, max(1, min(20705, most))), "D": D, "F": F,
                "act": rng.choice(["silu", "gelu"]), "train": train}
    D = _log_int(rng, 16, 8192)
    return {"op": op, "dtype": dtype, "M": _log_int(rng, 1, max(1, 206848 * 512 // D // (BYTES[dtype] // 2))), "D": D,
            "train": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs --
def _log_decay(H, device):
    # half-lives spread from one step to a few hundred
    e = torch.linspace(1.0, 8.0, H, device=device) if H > 1 else torch.tensor([5.0], device=device)
    return torch.log1p(-torch.exp2(-e))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).mul_(std).to(dtype)

    st = {"case": dict(case)}
    op = case["op"]
    if op in ("step", "attn"):
        B, H, Hk, dk, dv = (case[k] for k in ("B", "H", "Hk", "dk", "dv"))
        st["log_decay"] = _log_decay(H, dev)
        tok = (B,) if op == "step" else (B, case["T"])
        st["q"], st["k"], st["v"] = normal(*tok, H, dk), normal(*tok, Hk, dk), normal(*tok, Hk, dv)
        if op == "step":
            st["state"] = normal(B, H, dk, dv, dtype=torch.float32)
            st["active"] = (torch.rand(B, generator=g, device=dev) < 0.75) if case["masked"] else None
            return st
        st["state"] = normal(B, H, dk, dv, dtype=torch.float32) if case["state"] else None
        st["lengths"] = (torch.randint(0, case["T"] + 1, (B,), generator=g, device=dev, dtype=torch.int32)
                         if case["ragged"] else None)
        if case["train"]:
            st["do"] = normal(*tok, H, dv)
            st["dstate"] = normal(B, H, dk, dv, dtype=torch.float32)
            for k in ("q", "k", "v", "state"):
                if st[k] is not None:
                    st[k].requires_grad_(True)
        return st
    M, D = case["M"], case["D"]
    if op == "ff":
        F = case["F"]
        st["x"] = normal(M, D)
        st["wg"], st["wu"] = normal(F, D, std=D ** -0.5), normal(F, D, std=D ** -0.5)
        st["wd"] = normal(D, F, std=F ** -0.5)
        names = ("x", "wg", "wu", "wd")
        if case["train"]:
            st["dy"] = normal(M, D)
    else:
        st["x"], st["r"] = normal(M, D), normal(M, D, std=2.0)
        st["w"] = (1.0 + normal(D, std=0.1, dtype=torch.float32)).to(dt)
        names = ("x", "r", "w")
        if case["train"]:
            st["dy"], st["ds"] = normal(M, D), normal(M, D)
    if case["train"]:
        for k in names:
            st[k].requires_grad_(True)
    return st


# ------------------------------------------------------------- plain forms --
def _plain_step(st):
    c, S = st["case"], st["state"]
    G, scale = c["H"] // c["Hk"], c["dk"] ** -0.5
    q = st["q"].float()
    k = st["k"].float().repeat_interleave(G, dim=1)
    v = st["v"].float().repeat_interleave(G, dim=1)
    new = S * torch.exp(st["log_decay"])[:, None, None] + k[..., :, None] * v[..., None, :]
    o = scale * (q[..., :, None] * new).sum(dim=-2)
    if st["active"] is not None:
        on = st["active"][:, None, None]
        o = torch.where(on, o, 0.0)
        new = torch.where(on[..., None], new, S)
    S.copy_(new)
    return o.to(st["q"].dtype), S


def _plain_attn(q, k, v, log_decay, state, lengths):
    """Chunked: within a chunk by the masked product, between chunks by the
    decay from each chunk's end to each later chunk's start."""
    B, T, H, dk = q.shape
    dv, G, C = v.shape[-1], H // k.shape[2], min(PLAIN_CHUNK, q.shape[1])
    n = -(-T // C)
    dev, dt = q.device, q.dtype
    t = torch.arange(T, device=dev)
    live = (t < lengths[:, None])[..., None, None] if lengths is not None else torch.ones((), dtype=torch.bool, device=dev)
    q, k, v = (torch.where(live, x.float(), 0.0) for x in (q, k, v))
    k, v = k.repeat_interleave(G, dim=2), v.repeat_interleave(G, dim=2)
    # the final state, straight from its sum
    end = lengths[:, None] if lengths is not None else torch.full((1, 1), T, device=dev)
    back = torch.clamp(end - 1 - t, min=0)[..., None].float()  # (B or 1, T, 1)
    kd = k * torch.exp(back * log_decay)[..., None]
    final = torch.matmul(kd.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3))
    if state is not None:
        final = final + state * torch.exp(end[..., None].float() * log_decay[:, None])[..., None]

    def chunks(x):  # (B, H, n, C, d), zeros past T
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * C - T))
        return x.reshape(B, n, C, H, x.shape[-1]).permute(0, 3, 1, 2, 4)

    qc, kc, vc = chunks(q), chunks(k), chunks(v)
    i = torch.arange(C, device=dev)
    lag = (i[:, None] - i).float()
    decay = torch.where(lag >= 0, torch.exp(lag.clamp(min=0) * log_decay[:, None, None]), 0.0)  # (H, C, C)
    o = torch.matmul(torch.matmul(qc, kc.transpose(-1, -2)) * decay[:, None], vc)
    gi = torch.exp((i + 1).float() * log_decay[:, None])  # (H, C)
    gj = torch.exp((C - 1 - i).float() * log_decay[:, None])
    if n > 1:
        own_sum = torch.matmul((kc * gj[:, None, :, None]).transpose(-1, -2), vc)  # (B, H, n, dk, dv)
        m = torch.arange(n, device=dev)
        gap = (m[:, None] - 1 - m).float()
        between = torch.where(gap >= 0, torch.exp(gap.clamp(min=0) * (C * log_decay[:, None, None])), 0.0)
        start = torch.matmul(between, own_sum.reshape(B, H, n, dk * dv)).reshape(B, H, n, dk, dv)
    else:
        start = torch.zeros((B, H, n, dk, dv), device=dev)
    if state is not None:
        m = torch.arange(n, device=dev).float()
        start = start + state[:, :, None] * torch.exp(m * (C * log_decay[:, None]))[..., None, None]
    o = o + torch.matmul(qc * gi[:, None, :, None], start)
    o = o.permute(0, 2, 3, 1, 4).reshape(B, n * C, H, dv)[:, :T] * dk ** -0.5
    return o.to(dt), final


def _plain_act(x, act):
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))  # gelu


def _plain_ff(x, wg, wu, wd, act):
    xf = x.float()
    h = _plain_act(torch.matmul(xf, wg.float().t()), act) * torch.matmul(xf, wu.float().t())
    return torch.matmul(h, wd.float().t()).to(x.dtype)


def _plain_norm(x, r, w):
    s = x.float() + r.float()
    y = s * torch.rsqrt((s * s).mean(dim=-1, keepdim=True) + EPS) * w.float()
    return y.to(x.dtype), s.to(x.dtype)


def run(state):
    c = state["case"]
    op = c["op"]
    if own:
        from turbompc_amd import learning
    if op == "step":
        if own:
            o = learning.decay_attention_step(state["q"], state["k"], state["v"], state["log_decay"], state["state"],
                                              active=state["active"])
            return {"o": o, "state": state["state"]}
        o, S = _plain_step(state)
        return {"o": o, "state": S}
    train = c["train"]
    with torch.set_grad_enabled(train):
        if op == "attn":
            args = (state["q"], state["k"], state["v"], state["log_decay"], state["state"], state["lengths"])
            o, S = learning.decay_attention(*args) if own else _plain_attn(*args)
            out, of, given = {"o": o, "state": S}, (o, S), (state["do"], state["dstate"]) if train else ()
            names = [k for k in ("q", "k", "v", "state") if state[k] is not None]
        elif op == "ff":
            args = (state["x"], state["wg"], state["wu"], state["wd"], c["act"])
            y = learning.gated_feed_forward(*args) if own else _plain_ff(*args)
            out, of, given = {"y": y}, (y,), (state["dy"],) if train else ()
            names = ["x", "wg", "wu", "wd"]
        else:
            args = (state["x"], state["r"], state["w"])
            y, s = learning.rms_norm_residual(*args, eps=EPS) if own else _plain_norm(*args)
            out, of, given = {"y": y, "s": s}, (y, s), (state["dy"], state["ds"]) if train else ()
            names = ["x", "r", "w"]
        if train:
            grads = torch.autograd.grad(of, [state[k] for k in names], given)
            out = {k: t.detach() for k, t in out.items()}
            out.update({"d" + k: t for k, t in zip(names, grads)})
    return out


def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op in ("step", "attn"):
        B, H, Hk, dk, dv = (case[k] for k in ("B", "H", "Hk", "dk", "dv"))
        if op == "step":
            live = 0.75 if case["masked"] else 1.0  # idle vehicles' states stay where they are
            return {"bytes": live * B * H * 8 * dk * dv + B * e * (H * (dk + dv) + Hk * (dk + dv)),
                    "flops": live * B * H * 5 * dk * dv}
        tok = B * case["T"]
        live = tok * (0.5 if case["ragged"] else 1.0)  # rows past a history's end are written, not read
        S = B * H * dk * dv * 4
        nbytes = live * e * (H * dk + Hk * (dk + dv)) + tok * e * H * dv + S * (2 if case["state"] else 1)
        flops = live * H * 4 * dk * dv
        if case["train"]:
            nbytes += live * e * (H * dk + Hk * (dk + dv) + H * dv) + tok * e * (H * dk + Hk * (dk + dv))
            nbytes += S * (3 if case["state"] else 1)
            flops += live * H * 8 * dk * dv
        return {"bytes": nbytes, "flops": flops}
    M, D = case["M"], case["D"]
    if op == "ff":
        F = case["F"]
        nbytes, flops = e * (2 * M * D + 3 * D * F), 6.0 * M * D * F
        if case["train"]:
            nbytes += e * (3 * M * D + 6 * D * F)
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    nbytes, flops = e * (4 * M * D + D), 5.0 * M * D
    if case["train"]:
        nbytes += e * (4 * M * D + 2 * D)
        flops += 9.0 * M * D
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    """From the definitions in 64 bits: the recurrences step by step, the
    derivatives written out."""
    st = prepare(case, seed)
    f = {k: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t) for k, t in st.items()}
    op = case["op"]
    with torch.no_grad():
        if op in ("step", "attn"):
            return _exact_recurrence(case, f)
        if op == "ff":
            return _exact_ff(case, f)
        x, r, w = f["x"], f["r"], f["w"]
        s = x + r
        ms = s.pow(2).sum(-1, keepdim=True) / case["D"] + EPS
        out = {"y": s / ms.sqrt() * w, "s": s}
        if case["train"]:
            a = f["dy"] * w
            dx = a / ms.sqrt() - s * (a * s).sum(-1, keepdim=True) / (case["D"] * ms.pow(1.5)) + f["ds"]
            out.update(dx=dx, dr=dx, dw=(f["dy"] * s / ms.sqrt()).sum(0))
        return out


def _exact_ff(case, f):
    act = case["act"]
    g, u = f["x"] @ f["wg"].t(), f["x"] @ f["wu"].t()
    if act == "silu":
        sg = torch.sigmoid(g)
        a, da = g * sg, sg * (1.0 + g * (1.0 - sg))
    else:
        phi = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
        a, da = g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    out = {"y": (a * u) @ f["wd"].t()}
    if case["train"]:
        dh = f["dy"] @ f["wd"]
        dg, du = dh * u * da, dh * a
        out.update(dx=dg @ f["wg"] + du @ f["wu"], dwg=dg.t() @ f["x"], dwu=du.t() @ f["x"],
                   dwd=f["dy"].t() @ (a * u))
    return out


def _exact_recurrence(case, f):
    B, H, Hk, dk, dv = (case[k] for k in ("B", "H", "Hk", "dk", "dv"))
    step = case["op"] == "step"
    T = 1 if step else case["T"]
    # the recurrence takes about 0.1 ms a step and direction, more where the states are large
    if T * (3 if case.get("train") else 1) * max(1e-4, B * H * dk * dv * 8 * 6 / 3e12) > 18.0:
        return None
    G, scale = H // Hk, dk ** -0.5
    shape = (lambda x: x[:, None]) if step else (lambda x: x)
    q, k, v = (shape(f[n]) for n in ("q", "k", "v"))
    kh = torch.arange(H, device=q.device) // G
    gamma = torch.exp(f["log_decay"])[:, None, None]
    S = f["state"].clone() if f["state"] is not None else torch.zeros((B, H, dk, dv), dtype=torch.float64, device=q.device)
    if step:
        n = f["active"].long() if f["active"] is not None else torch.ones(B, dtype=torch.long, device=q.device)
    else:
        n = f["lengths"].long() if f["lengths"] is not None else torch.full((B,), T, device=q.device)
    whole = bool((n == T).all())
    train = bool(case.get("train"))
    o = torch.zeros((B, T, H, dv), dtype=torch.float64, device=q.device)
    dq = torch.zeros((B, T, H, dk), dtype=torch.float64, device=q.device) if train else None
    for t in range(T):
        new = torch.addcmul(S * gamma, k[:, t, kh, :, None], v[:, t, kh, None, :])
        on = (n > t)[:, None, None]
        S = new if whole else torch.where(on[..., None], new, S)
        ot = scale * torch.matmul(q[:, t, :, None, :], new)[..., 0, :]
        o[:, t] = ot if whole else torch.where(on, ot, 0.0)
        if train:
            d = scale * torch.matmul(new, f["do"][:, t, :, :, None])[..., 0]
            dq[:, t] = d if whole else torch.where(on, d, 0.0)
    out = {"o": o[:, 0] if step else o, "state": S}
    if not train:
        return out
    R = f["dstate"].clone()  # dL/d(state after step t), from what comes later
    dk_, dv_ = torch.zeros_like(k), torch.zeros_like(v)
    for t in range(T - 1, -1, -1):
        new = torch.addcmul(R, q[:, t, :, :, None], scale * f["do"][:, t, :, None, :])
        on = (n > t)[:, None, None]
        a = torch.matmul(new, v[:, t, kh, :, None])[..., 0]
        b = torch.matmul(k[:, t, kh, None, :], new)[..., 0, :]
        if not whole:
            a, b, new = torch.where(on, a, 0.0), torch.where(on, b, 0.0), torch.where(on[..., None], new * gamma, R)
        else:
            new = new * gamma
        dk_[:, t] = a.reshape(B, Hk, G, dk).sum(2)
        dv_[:, t] = b.reshape(B, Hk, G, dv).sum(2)
        R = new
    out.update(dq=dq, dk=dk_, dv=dv_)
    if f["state"] is not None:
        out["dstate"] = R
    return out
