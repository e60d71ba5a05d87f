"""The gated delta rule (turbompc_amd.learning) against its definition in 64 bits."""
import pytest
import torch

import learning_reference_delta as ref
from turbompc_amd import learning

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]


def inputs(B, T, heads, dk, dv, dtype, seed=0, state=True, lengths=None):
    """heads: (H, Hq, Hk, Hv)"""
    H, Hq, Hk, Hv = heads
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    k = r(B, T, Hk, dk)
    k = k / k.norm(dim=-1, keepdim=True)
    half = torch.linspace(1.0, 7.0, H) if H > 1 else torch.tensor([4.0])
    x = dict(q=r(B, T, Hq, dk).to(dtype), k=k.to(dtype), v=r(B, T, Hv, dv).to(dtype),
             g=torch.log1p(-torch.exp2(-half)) * torch.exp(0.5 * r(B, T, H)), beta=torch.sigmoid(r(B, T, H)).to(dtype),
             state=r(B, H, dk, dv) * dk ** -0.5 if state else None,
             lengths=torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None,
             do=r(B, T, H, dv).to(dtype), dstate=r(B, H, dk, dv))
    return {n: t.to(DEV) if t is not None else None for n, t in x.items()}


def forward(x, **kw):
    with torch.no_grad():
        return learning.delta_attention(x["q"], x["k"], x["v"], x["g"], x["beta"], x["state"], x["lengths"], **kw)


def check_forward(x, **kw):
    o, s = forward(x, **kw)
    want = ref.delta(x["q"], x["k"], x["v"], x["g"], x["beta"], x["state"], x["lengths"], **kw)
    ref.assert_within("o", o, want["o"], 2)
    ref.assert_within("state", s, want["state"], 1)
    return o, s


SHAPES = [  # B, T, (H, Hq, Hk, Hv), dk, dv
    (1, 1, (1, 1, 1, 1), 1, 1), (2, 5, (2, 2, 2, 2), 16, 16), (1, 16, (1, 1, 1, 1), 32, 32), (2, 17, (4, 4, 2, 2), 33, 57),
    (1, 63, (2, 1, 1, 2), 64, 64), (2, 64, (3, 3, 3, 3), 48, 80), (1, 65, (2, 2, 1, 1), 128, 32), (1, 130, (2, 2, 2, 2), 64, 128),
    (1, 200, (4, 1, 1, 4), 128, 128), (1, 333, (1, 1, 1, 1), 127, 96), (3, 97, (4, 2, 4, 1), 20, 128),
    (1, 64, (6, 2, 3, 6), 96, 24),
]
SHAPE_IDS = lambda s: "x".join(map(str, s)).replace(" ", "")  # noqa: E731


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=SHAPE_IDS)
def test_histories(shape, state, dtype):
    check_forward(inputs(*shape, dtype, seed=sum(shape[:2]), state=state))


LENGTHS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 80, 90, 300, -4]


@pytest.mark.parametrize("dtype", DTYPES)
def test_ragged_histories(dtype):
    """Lengths of zero, one, block and chunk ends, above T and below zero; what rows past a length hold
    is not read, and their outputs are zero."""
    x = inputs(len(LENGTHS), 90, (4, 4, 2, 2), 33, 40, dtype, seed=1, lengths=LENGTHS)
    want = check_forward(x)
    bad = dict(x)
    for n in ("q", "k", "v", "g", "beta"):
        bad[n] = x[n].clone()
        for b, L in enumerate(LENGTHS):
            bad[n][b, max(L, 0):] = float("nan")
    got = forward(bad)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for b, L in enumerate(LENGTHS):
        assert not bool(got[0][b, max(L, 0):].any())


def gates_at_their_ends(dk, dv, dtype):
    x = inputs(2, 150, (2, 2, 2, 2), dk, dv, dtype, seed=2)
    x["g"][0, 3], x["g"][0, 64], x["g"][0, 70:73], x["g"][1, 15:17] = (-float("inf"),) * 4
    x["g"][0, 20:60] = 0.0
    x["g"][1, 40], x["g"][1, 41], x["g"][1, 90] = -90.0, -1e4, -1e30
    x["beta"][0, 30:50], x["beta"][1, 30:50], x["beta"][1, 60:100] = 0.0, 1.0, 2.0
    x["k"][1, 100:140] = x["k"][1, 100:101]
    x["beta"][1, 100:140] = 1.0
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(32, 64), (128, 128)])
def test_gates_at_their_ends(dtype, dk, dv):
    """Decays of zero (-inf), of one, and far below what an exponential holds; rates of 0, 1 and 2; keys
    that repeat themselves."""
    check_forward(gates_at_their_ends(dk, dv, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_zero_keys_values_and_scale(dtype):
    x = inputs(1, 70, (2, 2, 2, 2), 32, 32, dtype, seed=3)
    x["k"][0, 10:30], x["v"][0, 5:8], x["q"][0, 40] = 0.0, 0.0, 0.0
    check_forward(x, scale=-0.7)
    o, s = forward(x, scale=0.0)
    assert not bool(o.any()) and bool(s.any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_views(dtype):
    """A fused projection's heads, expanded and transposed inputs give what their copies give."""
    H, d = 4, 32
    gen = torch.Generator().manual_seed(4)
    proj = torch.randn(2, 70, 3 * H * d + 2 * H, generator=gen).to(dtype).to(DEV) * 0.2
    q, k, v = (t.unflatten(-1, (H, d)) for t in proj[..., :3 * H * d].split(H * d, -1))
    beta = proj[..., 3 * H * d:3 * H * d + H]
    beta.copy_(torch.sigmoid(beta.float()))
    g = -torch.rand(H, 70, 2, generator=gen).to(DEV).permute(2, 1, 0)
    x = dict(q=q, k=k[:, :, :1].expand(-1, -1, H, -1), v=v.transpose(0, 1).contiguous().transpose(0, 1), g=g, beta=beta,
             state=torch.randn(1, H, d, d, generator=gen).to(DEV).expand(2, -1, -1, -1),
             lengths=torch.tensor([[60, 1], [70, 1]], dtype=torch.int32, device=DEV)[:, 0])
    want = forward({n: t.contiguous() for n, t in x.items()})
    for a, b in zip(forward(x), want):
        assert torch.equal(a, b)
    wide = torch.zeros(2, 70, H, 2 * d, dtype=dtype, device=DEV)
    wide[..., ::2] = q
    odd = torch.zeros(2 * 70 * H * d + 1, dtype=dtype, device=DEV)[1:].view(2, 70, H, d).copy_(q)  # one element off
    for y in (wide[..., ::2], odd):
        for a, b in zip(forward(dict(x, q=y)), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_windows_that_continue(dtype):
    """A history in windows, each from the state the last one left, ends in the whole one's state."""
    x = inputs(2, 150, (2, 2, 2, 2), 40, 24, dtype, seed=5)
    state, rows = x["state"], []
    for a, b in ((0, 37), (37, 38), (38, 150)):
        part = {n: x[n][:, a:b] for n in ("q", "k", "v", "g", "beta")}
        w, state = forward(dict(part, state=state, lengths=None))
        rows.append(w)
    want = ref.delta(x["q"], x["k"], x["v"], x["g"], x["beta"], x["state"])
    ref.assert_within("state", state, want["state"], 1)
    if dtype == torch.float32:  # the tolerance of bf16 is for blocks that begin at multiples of 16
        ref.assert_within("o", torch.cat(rows, 1), want["o"], 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_spoiled_values_reach_no_earlier_step(dtype, bad):
    x = inputs(3, 100, (2, 2, 2, 2), 32, 48, dtype, seed=6)
    o, s = forward(x)
    for n in ("q", "k", "v", "beta", "g"):
        if n == "g" and bad == -float("inf"):
            continue  # a decay of zero
        y = dict(x, **{n: x[n].clone()})
        if n in ("g", "beta"):
            y[n][1, 37, 1] = bad
        else:
            y[n][1, 37, 1, 7] = bad
        po, ps = forward(y)
        other = torch.tensor([0, 2], device=DEV)
        assert torch.equal(po[other], o[other]) and torch.equal(ps[other], s[other])
        assert torch.equal(po[1, :, 0], o[1, :, 0]) and torch.equal(ps[1, 0], s[1, 0])
        want = ref.delta(x["q"][1:2, :37], x["k"][1:2, :37], x["v"][1:2, :37], x["g"][1:2, :37], x["beta"][1:2, :37],
                         x["state"][1:2])["o"]
        ref.assert_within(n, po[1:2, :37], want, 2)  # a run made again step by step rounds less
        assert not bool(torch.isfinite(po[1, 37, 1]).all())
        if n == "q":
            assert torch.equal(ps, s) and bool(torch.isfinite(po[1, 38:]).all())


# ------------------------------------------------------------------- step --
def step_inputs(B, heads, dk, dv, dtype, seed):
    x = inputs(B, 1, heads, dk, dv, dtype, seed=seed)
    return {n: x[n][:, 0] if n not in ("state", "lengths", "dstate") else x[n] for n in x}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, (1, 1, 1, 1), 1, 1), (3, (4, 2, 2, 4), 33, 57), (2, (2, 2, 1, 1), 128, 128),
                                   (5, (3, 3, 3, 3), 128, 4), (2, (6, 2, 3, 6), 7, 128), (64, (4, 4, 4, 4), 32, 32)], ids=str)
def test_step(shape, dtype):
    B = shape[0]
    x = step_inputs(*shape, dtype, seed=7)
    active = torch.arange(B, device=DEV) % 3 != 1
    for mask in (None, active):
        state = x["state"].clone()
        o = learning.delta_attention_step(x["q"], x["k"], x["v"], x["g"], x["beta"], state, mask)
        lengths = None if mask is None else mask.int()
        want = ref.delta(*(x[n][:, None] for n in ("q", "k", "v", "g", "beta")), x["state"], lengths)
        ref.assert_within("o", o[:, None], want["o"], 2)
        ref.assert_within("state", state, want["state"], 1)
        if mask is not None:
            assert torch.equal(state[~mask], x["state"][~mask]) and not bool(o[~mask].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_walk_a_history(dtype):
    x = inputs(2, 40, (4, 2, 2, 4), 24, 40, dtype, seed=8)
    state = x["state"].clone()
    rows = [learning.delta_attention_step(*(x[n][:, t] for n in ("q", "k", "v", "g", "beta")), state) for t in range(40)]
    want = ref.delta(x["q"], x["k"], x["v"], x["g"], x["beta"], x["state"])
    ref.assert_within("o", torch.stack(rows, 1), want["o"], 2)
    ref.assert_within("state", state, want["state"], 1)


def test_step_idle_problems_are_not_read():
    x = step_inputs(3, (2, 2, 2, 2), 16, 16, torch.float32, seed=9)
    active = torch.tensor([True, False, True], device=DEV)
    state = x["state"].clone()
    bad = {n: x[n].clone() for n in ("q", "k", "v", "g", "beta")}
    for t in (*bad.values(), state):
        t[1] = float("nan")
    o = learning.delta_attention_step(*bad.values(), state, active)
    good = x["state"].clone()
    want = learning.delta_attention_step(*(x[n] for n in bad), good, active)
    assert torch.equal(o, want) and torch.equal(state[active], good[active]) and bool(torch.isnan(state[1]).all())
