"""What the gated delta rule rounds to bf16 (turbompc_amd.learning.delta_attention): its results, once, and nothing
else by fewer than two terms.

An error above half a step of the result (2^-8 of it) is at most that of operands with two terms of 8 bits, in units of
e^2 = 2^-16 of the products' magnitudes.  Rounded to nearest an operand of two terms is off by e^2, cut off by 2 e^2;
where both of a product have two, that of the second ones is left out: another e^2, or two where one of them is what a
cut of the first term left.  So, at most, a product has
  o:   the state or u, cut off, with q exact or with a score, cut off:                        2 + 2 = 4,
  dq:  do, exact, with the state: 1; the score M, cut off, made from e and do: 2 + 1 =            3,
  dk:  e with the state's gradient, y with the state: 1 + 1 + 2 = 4; M as above; N from y and e: 2 + 1 + 1 + 1 = 5.
The magnitudes are summed up over blocks of 32 steps for o, as they are in bf16, and chunks of 64 for dq and dk."""
import pytest
import torch

import learning_reference_delta as ref
from learning_reference import BF16, cpu64
from test_gpu_learning_delta import LENGTHS, SHAPE_IDS, SHAPES, forward, gates_at_their_ends, inputs
from test_gpu_learning_delta_gradients import NAMES, run

pytestmark = pytest.mark.gpu
DTYPE = torch.bfloat16


def bounds(x, monkeypatch, scale=None):
    """{"o", "dq", "dk"}: (value, tolerance, limit) as above."""
    monkeypatch.setattr(ref, "BLOCK", 32)
    q, k, v, g, beta = (x[n] for n in NAMES[:5])
    B, T, H = g.shape
    n = torch.full((B,), T) if x["lengths"] is None else x["lengths"].cpu().long().clamp(0, T)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    live = (torch.arange(T) < n[:, None])[..., None]
    f = [torch.where(live[..., None], cpu64(z).repeat_interleave(H // z.shape[2], 2), 0.0) for z in (q, k, v)]
    g, beta = torch.where(live, cpu64(g), 0.0), torch.where(live, cpu64(beta), 0.0)
    do = torch.where(live[..., None], cpu64(x["do"]), 0.0)
    y = ref._loop(*f, g, beta, cpu64(x["state"]), n, scale, do, cpu64(x["dstate"]))
    mo, mq, mk = ref._magnitudes(y, f[0], f[1], g, beta, scale, do)
    out = {}
    for name, value, mag, heads, units, chain in (("o", y["o"], mo, H, 4, 3), ("dq", y["dq"], mq, q.shape[2], 3, 6),
                                                  ("dk", y["dk"], mk, k.shape[2], 5, 6)):
        value, mag = (z.reshape(B, T, heads, H // heads, -1).sum(3) for z in (value, mag))
        # 1.02: what is of third order, and the exponentials' own error
        out[name] = value, BF16 * value.abs() + 1.02 * units * BF16 ** 2 * mag, ref.norm_limit(T, q.shape[-1], v.shape[-1], chain), None
    return out


def check(x, monkeypatch):
    got, want = run(x), bounds(x, monkeypatch)
    for n in want:
        ref.assert_within(n, got[n], want[n], 2)


@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("shape", [*SHAPES, (1, 600, (2, 2, 2, 2), 32, 32), (1, 1100, (1, 1, 1, 1), 64, 128), (64, 12, (4, 4, 4, 4), 16, 16)],
                         ids=SHAPE_IDS)
def test_results_are_rounded_once(shape, state, monkeypatch):
    x = inputs(*shape, DTYPE, seed=sum(shape[:2]) + 200, state=state)
    if not state:
        x["dstate"] = None
    check(x, monkeypatch)


def test_ragged_histories(monkeypatch):
    check(inputs(len(LENGTHS), 90, (4, 4, 2, 2), 33, 40, DTYPE, seed=202, lengths=LENGTHS), monkeypatch)


@pytest.mark.parametrize("dk,dv", [(32, 64), (128, 128)])
def test_gates_at_their_ends(dk, dv, monkeypatch):
    check(gates_at_their_ends(dk, dv, DTYPE), monkeypatch)


def test_outputs_of_windows_that_continue(monkeypatch):
    """Blocks begin where a window does: the outputs of each window from the state that the last one left."""
    x = inputs(2, 150, (2, 2, 2, 2), 40, 24, DTYPE, seed=205)
    state = x["state"]
    whole = bounds(x, monkeypatch)["o"][0]
    for a, b in ((0, 37), (37, 38), (38, 150)):
        part = dict(x, state=state, lengths=None, **{n: x[n][:, a:b] for n in ("q", "k", "v", "g", "beta", "do")})
        value, tol, limit, _ = bounds(part, monkeypatch)["o"]
        o, state = forward(part)
        ref.assert_within("o", o, (value, tol, limit, None), 2)
        # against the whole history, whose state at the window's start is off by its own limit more
        ref.assert_within("o", o, (whole[:, a:b], tol, limit + ref.norm_limit(b, 40, 24, 6), None), 2)
