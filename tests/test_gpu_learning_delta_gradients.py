"""The gated delta rule's gradients (turbompc_amd.learning) against the formulas in 64 bits and against
differences."""
import pytest
import torch

import learning_reference as base
import learning_reference_delta as ref
from test_gpu_learning_delta import DTYPES, LENGTHS, SHAPE_IDS, SHAPES, gates_at_their_ends, inputs
from test_gpu_learning_gradients import check_differences, weighted
from turbompc_amd import learning

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("q", "k", "v", "g", "beta", "state")
AXES = {"dq": 2, "dk": 2, "dv": 2, "dg": 2, "dbeta": 2, "dstate": 1, "o": 2, "state": 1}


def run(x, **kw):
    leaf = {n: x[n].detach().requires_grad_(True) for n in NAMES if x[n] is not None}
    o, s = learning.delta_attention(*(leaf.get(n) for n in NAMES), x["lengths"], **kw)
    given = [(t, g) for t, g in ((o, x["do"]), (s, x["dstate"])) if g is not None]
    grads = torch.autograd.grad([t for t, _ in given], list(leaf.values()), [g for _, g in given])
    return {"o": o.detach(), "state": s.detach(), **{"d" + n: g for n, g in zip(leaf, grads)}}


def check(x, **kw):
    got = run(x, **kw)
    do = x["do"] if x["do"] is not None else torch.zeros(x["g"].shape + x["v"].shape[-1:], dtype=x["q"].dtype)
    want = ref.delta(*(x[n] for n in NAMES), x["lengths"], kw.get("scale"), do, x["dstate"])
    for n in got:
        ref.assert_within(n, got[n], want[n], AXES[n])
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=SHAPE_IDS)
def test_gradients(shape, state, dtype):
    x = inputs(*shape, dtype, seed=sum(shape[:2]) + 100, state=state)
    if not state:
        x["dstate"] = None
    check(x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_over_several_stretches(dtype):
    """Histories longer than the stretches in which log_decay's gradient is summed."""
    check(inputs(1, 600, (2, 2, 2, 2), 32, 32, dtype, seed=101))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 1100, (1, 1, 1, 1), 32, 48), (1, 1300, (2, 1, 2, 2), 64, 40), (3, 1030, (1, 1, 1, 1), 20, 100)],
                         ids=SHAPE_IDS)
def test_long_histories_in_runs(shape, dtype):
    """Few heads of many steps: cut into runs, forwards and backwards, ragged (a run that is not reached, one
    that ends inside, lengths of zero and one)."""
    B, T = shape[:2]
    check(inputs(*shape, dtype, seed=109))
    x = inputs(*shape, dtype, seed=110, lengths=[T - 300, 1, 0][:B] if B != 2 else [513, T])
    want = check(x)
    for b, L in enumerate(x["lengths"].tolist()):
        for n in ("o", "dq", "dk", "dv", "dg", "dbeta"):
            assert not bool(want[n][b, L:].any()), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1100, (1, 1, 1, 1), 128, 128), (1, 1050, (2, 1, 1, 2), 100, 24), (1, 2299, (64, 32, 64, 64), 8, 8)],
                         ids=SHAPE_IDS)
def test_runs_of_other_widths_and_lengths(shape, dtype):
    """Heads of 128 and of up to 32, whose runs go by other columns a workgroup; runs of two stretches, the
    last one of one."""
    check(inputs(*shape, dtype, seed=127))


def test_spoiled_values_in_runs():
    """A value that is not finite in one run of several: earlier runs' outputs stay, later ones are spoiled."""
    x = inputs(1, 1300, (2, 2, 2, 2), 32, 32, torch.float32, seed=111)
    with torch.no_grad():
        o, s = learning.delta_attention(*(x[n] for n in NAMES))
        for n in ("k", "v"):
            y = dict(x, **{n: x[n].clone()})
            y[n][0, 700, 1, 3] = float("nan")
            po, ps = learning.delta_attention(*(y[m] for m in NAMES))
            assert torch.equal(po[:, :, 0], o[:, :, 0]) and torch.equal(ps[:, 0], s[:, 0])
            want = ref.delta(*(x[m][:, :700] for m in NAMES[:5]), x["state"])["o"]
            ref.assert_within(n, po[:, :700], want, 2)
            cols = slice(3, 4) if n == "v" else slice(None)
            assert bool(torch.isnan(po[0, 700:, 1, cols]).all()) and bool(torch.isnan(ps[0, 1, :, cols]).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_ragged_gradients(dtype):
    x = inputs(len(LENGTHS), 90, (4, 4, 2, 2), 33, 40, dtype, seed=102, lengths=LENGTHS)
    want = check(x)
    bad = dict(x)
    for n in ("q", "k", "v", "g", "beta", "do"):
        bad[n] = x[n].clone()
        for b, L in enumerate(LENGTHS):
            bad[n][b, max(L, 0):] = float("nan")
    got = run(bad)
    for n in got:
        assert torch.equal(got[n], want[n]), n
    for b, L in enumerate(LENGTHS):
        for n in ("dq", "dk", "dv", "dg", "dbeta"):
            assert not bool(got[n][b, max(L, 0):].any()), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(32, 64), (128, 128)])
def test_gradients_with_gates_at_their_ends(dk, dv, dtype):
    x = gates_at_their_ends(dk, dv, dtype)
    got = check(x)
    assert not bool(got["dg"][torch.isinf(x["g"])].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_one_output_alone(dtype):
    x = inputs(2, 40, (2, 2, 2, 2), 24, 40, dtype, seed=103)
    check(dict(x, do=None))
    check(dict(x, dstate=None))
    check(dict(x, state=None), scale=-0.3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_shared_heads_are_their_sums(dtype):
    """Each of q, k and v shared alone, against the sum over repeated heads."""
    for heads in ((4, 2, 4, 4), (4, 4, 1, 4), (6, 6, 6, 3)):
        x = inputs(2, 50, heads, 32, 24, dtype, seed=104)
        got = check(x)
        H = heads[0]
        full = {n: x[n].repeat_interleave(H // x[n].shape[2], 2) for n in ("q", "k", "v")}
        whole = run(dict(x, **full))
        assert torch.equal(got["o"], whole["o"]) and torch.equal(got["dg"], whole["dg"])
        for n in ("q", "k", "v"):
            if x[n].shape[2] == H:
                assert torch.equal(got["d" + n], whole["d" + n]), n


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_through_views(dtype):
    x = inputs(2, 70, (2, 2, 2, 2), 32, 48, dtype, seed=105)
    want = run(x)
    wide = torch.zeros(2, 70, 2, 100, dtype=dtype, device=DEV)
    wide[..., 1:49] = x["do"]
    proj = torch.cat([x["q"], x["k"]], -1)
    got = run(dict(x, q=proj[..., :32], k=proj[..., 32:], v=x["v"].transpose(0, 1).contiguous().transpose(0, 1),
                   g=x["g"].permute(2, 1, 0).contiguous().permute(2, 1, 0), do=wide[..., 1:49]))
    for n in want:
        assert torch.equal(got[n], want[n]), n
    ones = run(dict(x, do=torch.ones((), dtype=dtype, device=DEV).expand(x["do"].shape)))
    full = run(dict(x, do=torch.ones_like(x["do"])))
    for n in ones:
        assert torch.equal(ones[n], full[n]), n


def test_equal_inputs_give_equal_bits():
    x = inputs(3, 150, (4, 2, 1, 4), 64, 64, torch.bfloat16, seed=106)
    first = run(x)
    for _ in range(3):
        again = run(x)
        for n in first:
            assert torch.equal(first[n], again[n]), n


@pytest.mark.parametrize("shape", [(2, 50, (4, 4, 2, 2), 24, 40), (1, 70, (1, 1, 1, 1), 128, 128)], ids=SHAPE_IDS)
def test_differences(shape):
    """Differences of the outputs in fp32 in each input, against the gradients.  The widths are those at which
    the bound, which the 64-bit formula alone gives, is under 4% (decays of several heads differ more in size)."""
    x = inputs(*shape, torch.float32, seed=107)
    got = run(x)
    full = ref.delta(*(x[n] for n in NAMES), None, None, x["do"], x["dstate"])
    grads = [x["do"], x["dstate"]]
    T, dk, dv = shape[1], shape[3], shape[4]

    def ours(n, v):
        z = dict(x, **{n: v})
        return weighted(learning.delta_attention(*(z[m] for m in NAMES)), grads)

    def formula(n, v):
        z = dict(x, **{n: v.float()})
        z = {m: (z[m].double() if m != n else v) for m in NAMES}
        out = ref.delta(*(z[m] for m in NAMES), x["lengths"])
        return weighted([out["o"][0], out["state"][0]], grads)

    # the outputs' rounding in the norm, against the weights' norm
    out = ref.delta(*(x[n] for n in NAMES))
    rounding = sum(ref.norm_limit(T, dk, dv, 3) * float(out[k][0].norm()) * float(base.cpu64(w).norm())
                   for k, w in zip(("o", "state"), grads)) / 8  # the units themselves, not eight times

    for n, h in (("q", 2.0), ("k", 0.3), ("v", 2.0), ("state", 2.0), ("beta", 1.0), ("g", 0.3 if shape[2][0] > 1 else 0.5)):
        check_differences(lambda v: ours(n, v), lambda v: formula(n, v), lambda v: rounding, x[n], got["d" + n],
                          full["d" + n][0], h, 108)


def test_more_chunks_than_a_row_of_workgroups():
    """Past 2^22 chunks the gradients' launch has rows of workgroups; the last problems are those of a
    call of their own."""
    B, T, H, d = (1 << 20) + 3, 65, 2, 4
    gen = torch.Generator(device=DEV).manual_seed(3)
    normal = lambda *s: torch.randn(s, generator=gen, device=DEV, dtype=torch.bfloat16)  # noqa: E731
    x = {n: normal(B, T, H, d) for n in "qkv"}
    x["g"] = -0.1 * torch.rand((B, T, H), generator=gen, device=DEV)
    x["beta"] = torch.rand((B, T, H), generator=gen, device=DEV).bfloat16()
    do = normal(B, T, H, d)

    def grads(b0):
        z = [x[n][b0:].detach().requires_grad_(True) for n in ("q", "k", "v", "g", "beta")]
        o, _ = learning.delta_attention(*z)
        return torch.autograd.grad(o, z, do[b0:])

    whole, part = grads(0), grads(B - 300)
    for name, got, want in zip(("q", "k", "v", "g", "beta"), whole, part):
        assert torch.equal(got[-300:], want), name
    del whole, part
    torch.cuda.empty_cache()
