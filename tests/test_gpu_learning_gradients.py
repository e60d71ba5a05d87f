"""Gradients of the history model's operators in fp32 against differences of their own outputs, and
errors in the norm against the formulas in 64 bits.

A direction is the sign of the formula's gradient over a random half of the entries, so that the
derivative along it is the sum of their magnitudes: a gradient that is zero, half, of the
other sign or wrong in a block is far outside.  The quotient is extrapolated from widths h and h / 2, which
leaves an error of 3 / h times the outputs' rounding (bounded elementwise at magnitudes as large as
the widths make them, weighted with the outputs' gradient) and the truncation, taken from the same
quotient in 64 bits; together at most 4% of the derivative, or the test says that it cannot tell.
"""
import pytest
import torch

import learning_reference as ref
import test_gpu_learning_attention as attention
import test_gpu_learning_blocks as blocks
from turbompc_amd import learning

pytestmark = pytest.mark.gpu


def directions(grad, scale, seed):
    gen = torch.Generator().manual_seed(seed)
    for _ in range(3):
        yield torch.sign(grad) * (torch.rand(grad.shape, generator=gen) < 0.5) * scale


def quotient(loss, x, d, h):
    at = lambda t: loss(x + t * d.to(x))  # noqa: E731
    wide, narrow = (at(h) - at(-h)) / (2 * h), (at(h / 2) - at(-h / 2)) / h
    return (4 * narrow - wide) / 3


def check_differences(loss, loss64, noise, x, got, want, h, seed):
    """loss, loss64: of the operator and of the formula, noise: the bound on the first's rounding, as
    functions of x; got, want: the gradients at x."""
    want = ref.cpu64(want)
    x64 = ref.cpu64(x)
    size = float(x64.std())
    rounding = 3 / h * noise((x.abs() + h * size) * torch.where(x < 0, -1.0, 1.0))
    for d in directions(want, size, seed):
        exact = float((want * d).sum())
        tol = rounding + abs(quotient(loss64, x64, d, h) - exact)
        assert tol < 0.04 * abs(exact), ("no test: the bound is too wide", tol, exact)
        ours = float((ref.cpu64(got) * d).sum())
        assert abs(quotient(loss, x, d, h) - ours) <= tol, (quotient(loss, x, d, h), ours, exact, tol)


def weighted(out, weights):
    return sum(float((ref.cpu64(o) * ref.cpu64(w)).sum()) for o, w in zip(out, weights))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_feed_forward_differences(act):
    x = blocks.ff_inputs(60, 48, 80, 48, torch.float32, seed=31)
    got = blocks.ff_run(x, act)
    names = ("x", "wg", "wu", "wd")
    want = ref.feed_forward(*(x[n] for n in names), act, x["dy"])
    for i, n in enumerate(names):
        ours = lambda v: weighted([learning.gated_feed_forward(*(v if m == n else x[m] for m in names), act)], [x["dy"]])  # noqa: E731
        formula = lambda v: ref.feed_forward(*(v if m == n else x[m] for m in names), act)["y"]  # noqa: E731
        check_differences(ours, lambda v: weighted([formula(v)[0]], [x["dy"]]),
                          lambda v: weighted([formula(v)[1]], [x["dy"].abs()]), x[n], got["d" + n], want["d" + n][0], 0.4,
                          32 + i)


def test_norm_differences():
    x = blocks.norm_inputs(20, 64, torch.float32, seed=33)
    got = blocks.norm_run(x)
    want = ref.norm(x["x"], x["r"], x["w"], 1e-6, x["dy"], x["ds"])

    def ours(n, v):
        z = dict(x, **{n: v})
        return weighted(learning.rms_norm_residual(z["x"], z["r"], z["w"]), [x["dy"], x["ds"]])

    def formula(n, v, which):
        z = dict(x, **{n: v})
        out = ref.norm(z["x"], z["r"], z["w"], 1e-6)
        return weighted([out[k][which] for k in ("y", "s")], [x[k].abs() if which else x[k] for k in ("dy", "ds")])

    for n, g in (("x", "dx"), ("r", "dx"), ("w", "dw")):
        check_differences(lambda v: ours(n, v), lambda v: formula(n, v, 0), lambda v: formula(n, v, 1), x[n], got["d" + n],
                          want[g][0], 0.4, 34)


@pytest.mark.parametrize("shape", [(2, 50, 4, 2, 24, 40), (1, 70, 1, 1, 128, 128)], ids=lambda s: "x".join(map(str, s)))
def test_attention_differences(shape):
    x = attention.inputs(*shape, torch.float32, seed=35)
    got = attention.run(x)
    full = ref.attention(x["q"], x["k"], x["v"], x["g"], x["state"], None, None, x["do"], x["dstate"])
    grads = [x["do"], x["dstate"]]

    def ours(n, v):
        z = dict(x, **{n: v})
        return weighted(learning.decay_attention(z["q"], z["k"], z["v"], z["g"], z["state"]), grads)

    def formula(n, v, which):
        z = dict(x, **{n: v})
        out = ref.attention(z["q"], z["k"], z["v"], z["g"], z["state"])
        out = attention.bounds(z, out, torch.float32) if which else out
        return weighted([out[k][which] for k in ("o", "state")], [w.abs() for w in grads] if which else grads)

    for n in ("q", "k", "v", "state"):
        check_differences(lambda v: ours(n, v), lambda v: formula(n, v, 0), lambda v: formula(n, v, 1), x[n], got["d" + n],
                          full["d" + n][0], 2.0, 36)


def assert_close_in_norm(name, got, value, n):
    """fp32 sums of n terms, one after another: their roundings are independent of each other, so the
    whole differs by about sqrt(n) units of its norm, a chain of three by less than twice that; eight
    times is allowed.  Operands rounded to bf16 would differ by 2^-9 or more."""
    got = ref.cpu64(got)
    limit = 8 * (n + 16) ** 0.5 * ref.F32
    assert limit < 2.0 ** -12
    assert float((got - value).norm()) <= limit * float(value.norm()), (name, float((got - value).norm() / value.norm()))


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("shape", [(64, 256, 683, 256), (129, 129, 130, 131), (300, 520, 260, 520), (1500, 40, 72, 40)],
                         ids=lambda s: "x".join(map(str, s)))
def test_feed_forward_fp32_norms(shape, act):
    x = blocks.ff_inputs(*shape, torch.float32, seed=37)
    got = blocks.ff_run(x, act)
    for k, (v, _) in ref.feed_forward(x["x"], x["wg"], x["wu"], x["wd"], act, x["dy"]).items():
        assert_close_in_norm(k, got[k], v, max(shape))


@pytest.mark.parametrize("shape", [(2, 130, 4, 2, 64, 48), (1, 200, 1, 1, 127, 127), (1, 1100, 2, 1, 128, 128)],
                         ids=lambda s: "x".join(map(str, s)))
def test_attention_fp32_norms(shape):
    x = attention.inputs(*shape, torch.float32, seed=38)
    got = attention.run(x)
    want = ref.attention(x["q"], x["k"], x["v"], x["g"], x["state"], None, None, x["do"], x["dstate"])
    for k, (v, _) in want.items():
        assert_close_in_norm(k, got[k], v, shape[1] + shape[4] + shape[5])


@pytest.mark.parametrize("M,D", [(70, 1000), (6000, 24), (9, 2049)])
def test_norm_fp32_norms(M, D):
    x = blocks.norm_inputs(M, D, torch.float32, seed=39)
    got = blocks.norm_run(x)
    for k, (v, _) in ref.norm(x["x"], x["r"], x["w"], 1e-6, x["dy"], x["ds"]).items():
        assert_close_in_norm(k, got[k], v, max(M, D))
