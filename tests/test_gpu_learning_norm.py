"""The layer norm with the residual's addition and dropout (turbompc_amd.learning) against their
definitions in 64 bits."""
import pytest
import torch

import learning_reference as base
import learning_reference_blocks as ref
from test_gpu_learning_gradients import check_differences, weighted
from turbompc_amd import learning

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]
KEY = (-0x123456789ABCDEF, 41)


def key(seed=KEY[0], step=KEY[1]):
    return torch.tensor([seed, step], device=DEV)


# ---------------------------------------------------------------- dropout --
def dropped(x, p, k, call):
    """The expected values of dropout on the CPU: fp32 products, rounded to x's type."""
    M, D = x.numel() // x.shape[-1], x.shape[-1]
    mask, f = ref.kept(M, D, p, k, call)
    v = (x.detach().cpu().float().reshape(M, D) * torch.tensor(f, dtype=torch.float32)).to(x.dtype)
    return torch.where(mask, v, torch.zeros((), dtype=x.dtype)).reshape(x.shape)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (7,), (3, 7), (64, 256), (2, 3, 1001), (1000, 12), (2, 20003), (70000, 3)],
                         ids=str)
def test_dropout(shape, dtype):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV).requires_grad_(True)
    dy = torch.randn(shape, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    for p, call in ((0.1, 0), (0.5, 2 ** 32 - 1)):
        y = learning.dropout(x, p, key(), call)
        assert torch.equal(y.detach().cpu(), dropped(x, p, KEY, call))
        dx, = torch.autograd.grad(y, x, dy)
        assert torch.equal(dx.cpu(), dropped(dy, p, KEY, call))
        with torch.no_grad():
            assert torch.equal(learning.dropout(x, p, key(), call), y)


@pytest.mark.parametrize("k", [(0, 0), (2 ** 63 - 1, 2 ** 32 - 1), (-1, -1), (5, 2 ** 32 + 5), (2 ** 40, 2 ** 62)], ids=str)
def test_dropout_keys(k):
    x = torch.randn(33, 70, generator=torch.Generator().manual_seed(3)).to(DEV)
    for call in (0, 9):
        assert torch.equal(learning.dropout(x, 0.3, key(*k), call).cpu(), dropped(x, 0.3, k, call))


def test_dropout_probabilities():
    """p is taken to the nearest 2^-16; what is dropped is zero whatever it holds; p = 0 is x."""
    x = torch.ones(257, 512, device=DEV)
    for p in (2.0 ** -16, 2.0 ** -18, 1.0 - 2.0 ** -16, 0.7):
        assert torch.equal(learning.dropout(x, p, key(), 1).cpu(), dropped(x, p, KEY, 1))
    assert learning.dropout(x, 0.0) is x and learning.dropout(x, 0.0, key()) is x
    share = float((learning.dropout(x, 0.25, key()) > 0).double().mean())
    # a binomial share of n = 131584 has a deviation of sqrt(0.1875 / n) = 1.2e-3: six of them
    assert abs(share - 0.75) < 7.2e-3
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device=DEV).repeat(40)
    y = learning.dropout(bad, 0.5, key())
    mask = ref.kept(1, 120, 0.5, KEY, 0)[0][0]
    assert bool((y.cpu()[~mask] == 0).all()) and not bool(torch.isfinite(y.cpu()[mask]).any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_goes_by_place_not_by_strides(dtype):
    wide = torch.randn(6, 5, 90, generator=torch.Generator().manual_seed(4)).to(dtype).to(DEV)
    for x in (wide[..., 3:44], wide.transpose(0, 1), wide[:, 2], wide[::2, ::3], wide[:, :, ::2], wide[:1].expand(4, -1, -1),
              wide.transpose(1, 2), wide[..., 0]):
        assert torch.equal(learning.dropout(x, 0.4, key(), 2).cpu(), dropped(x, 0.4, KEY, 2))
    empty = torch.zeros((0, 8), dtype=dtype, device=DEV, requires_grad=True)
    y = learning.dropout(empty, 0.4, key())
    y.sum().backward()
    assert y.shape == (0, 8) and empty.grad.shape == (0, 8)


def test_dropout_wide_launches():
    """More pieces than one launch's 32-bit indexes count are no matter of the values: here with rows
    of the largest width, against the same rows' first columns."""
    x = torch.ones(2, 1 << 24, dtype=torch.bfloat16, device=DEV)
    y = learning.dropout(x, 0.5, key(), 6)
    assert torch.equal(y[:, :4096].cpu(), dropped(x[:, :4096], 0.5, KEY, 6))
    end = ref.philox(((1 << 21) - 1, 1, 6, KEY[1]), (KEY[0] % 2 ** 32, (KEY[0] >> 32) % 2 ** 32))
    bits = [h for w in end for h in (int(w) & 0xFFFF, int(w) >> 16)]
    assert (y[1, -8:].cpu() > 0).tolist() == [b >= 32768 for b in bits]


# ------------------------------------------------------------- layer norm --
def norm_inputs(M, D, dtype, seed=0, offset=0.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(s, generator=gen) * std)  # noqa: E731
    return {k: t.to(dtype).to(DEV) for k, t in dict(x=r(M, D) + offset, r=r(M, D, std=2.0), w=1 + r(D, std=0.2), b=r(D),
                                                    dy=r(M, D), ds=r(M, D)).items()}


def norm_run(x, eps=1e-5, p=0.0, k=None, call=0):
    leaf = {n: x[n].detach().requires_grad_(True) for n in ("x", "r", "w", "b") if x[n] is not None}
    y, s = learning.layer_norm_residual(leaf["x"], leaf.get("r"), leaf["w"], leaf.get("b"), eps, p, k, call)
    given = [(o, g) for o, g in ((y, x["dy"]), (s, x["ds"])) if g is not None]
    grads = torch.autograd.grad([o for o, _ in given], list(leaf.values()), [g for _, g in given], allow_unused=True)
    return {"y": y.detach(), "s": s.detach(), **{"d" + n: g for n, g in zip(leaf, grads)}}


def check(x, got, eps=1e-5, p=0.0, k=None, call=0):
    want = ref.layer_norm(x["x"], x["r"], x["w"], x["b"], eps, x["dy"], x["ds"], p, k, call)
    for n in got:
        base.assert_within(n, got[n], *want[n])


NORM = [(1, 1), (3, 7), (5, 64), (7, 129), (4, 512), (3, 1000), (2, 1024), (2, 2047), (3, 2056), (2, 4097), (3, 8192),
        (5000, 72), (1300, 1024)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("shape", NORM, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm(shape, p, dtype):
    x = norm_inputs(*shape, dtype, seed=sum(shape))
    got = norm_run(x, p=p, k=key(), call=5)
    assert set(got) == {"y", "s", "dx", "dr", "dw", "db"}
    check(x, got, p=p, k=KEY, call=5)
    with torch.no_grad():  # without the statistics: the same numbers
        y, s = learning.layer_norm_residual(x["x"], x["r"], x["w"], x["b"], dropout=p, key=key(), call=5)
    assert torch.equal(y, got["y"]) and torch.equal(s, got["s"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("without", ["r", "b", "rb", "ds", "rbds"])
def test_layer_norm_without_some_inputs(without, dtype):
    for p in (0.0, 0.2):
        x = norm_inputs(9, 200, dtype, seed=7)
        for n in ("r", "b"):
            if n in without.replace("ds", ""):
                x[n] = None
        if "ds" in without:
            x["ds"] = None
        got = norm_run(x, p=p, k=key(), call=1)
        check(x, got, p=p, k=KEY, call=1)


def test_layer_norm_gradient_of_the_sum_alone():
    x = norm_inputs(9, 200, torch.float32, seed=8)
    got = norm_run(dict(x, dy=None), p=0.2, k=key())
    mask, f = ref.kept(9, 200, 0.2, KEY, 0)
    assert torch.equal(got["dr"], x["ds"]) and not bool(got["dw"].any()) and not bool(got["db"].any())
    assert torch.equal(got["dx"].cpu(), torch.where(mask, x["ds"].cpu() * f, torch.zeros(())))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_of_rows_far_from_zero_and_of_equal_values(dtype):
    """The mean is subtracted before the squares are summed, so a mean of a thousand deviations costs
    its own rounding and no more; a constant row has no deviation, and eps alone is left."""
    x = norm_inputs(20, 300, dtype, seed=9, offset=1000.0)
    check(x, norm_run(x, p=0.1, k=key()), p=0.1, k=KEY)
    c = torch.full((4, 256), 3.0, dtype=dtype, device=DEV)
    y, s = learning.layer_norm_residual(c, None, torch.ones(256, dtype=dtype, device=DEV))
    assert torch.equal(s, c) and not bool(y.any())


def test_layer_norm_dropout_is_dropouts():
    """d(x) of the norm has dropout's mask, in whatever row form it is made."""
    for D in (5, 100, 700, 3000, 8192):
        x = torch.randn(3, D, generator=torch.Generator().manual_seed(D)).to(DEV)
        s = learning.layer_norm_residual(x, None, torch.ones(D, device=DEV), dropout=0.5, key=key(), call=8)[1]
        assert torch.equal(s, learning.dropout(x, 0.5, key(), 8))


def test_layer_norm_strides_and_leading_axes():
    x = norm_inputs(24, 40, torch.bfloat16, seed=10)
    wide = torch.zeros((2, 12, 90), dtype=torch.bfloat16, device=DEV)
    wide[..., 3:43] = x["x"].view(2, 12, 40)
    want = norm_run(x, p=0.2, k=key())
    three = {n: x[n].view(2, 12, 40) for n in ("r", "dy", "ds")}
    got = norm_run(dict(x, **three, x=wide[..., 3:43], w=torch.stack([x["w"]] * 2, 1)[:, 0]), p=0.2, k=key())
    for n in want:
        assert torch.equal(got[n].reshape(want[n].shape), want[n]), n


def test_layer_norm_spoiled_rows_stay_alone():
    x = norm_inputs(40, 72, torch.float32, seed=11)
    want = norm_run(x)
    for v in (float("nan"), float("inf")):
        bad = dict(x, x=x["x"].clone())
        bad["x"][7, 5] = v
        got = norm_run(bad)
        rows = torch.arange(40, device=DEV) != 7
        for n in ("y", "s", "dx", "dr"):
            assert torch.equal(got[n][rows], want[n][rows]), n
        assert bool(torch.isnan(got["y"][7]).all())


def test_layer_norm_of_no_rows():
    x = norm_inputs(0, 24, torch.bfloat16)
    got = norm_run(x, p=0.1, k=key())
    assert got["y"].shape == (0, 24) and not bool(got["dw"].any()) and not bool(got["db"].any())


def test_layer_norm_differences():
    x = norm_inputs(20, 64, torch.float32, seed=12)
    got = norm_run(x, p=0.25, k=key(), call=3)
    want = ref.layer_norm(x["x"], x["r"], x["w"], x["b"], 1e-5, x["dy"], x["ds"], 0.25, KEY, 3)

    def ours(n, v):
        z = dict(x, **{n: v})
        return weighted(learning.layer_norm_residual(z["x"], z["r"], z["w"], z["b"], 1e-5, 0.25, key(), 3), [x["dy"], x["ds"]])

    def formula(n, v, which):
        z = dict(x, **{n: v})
        out = ref.layer_norm(z["x"], z["r"], z["w"], z["b"], 1e-5, p=0.25, key=KEY, call=3)
        return weighted([out[k][which] for k in ("y", "s")], [x[k].abs() if which else x[k] for k in ("dy", "ds")])

    for n in ("x", "r", "w", "b"):
        check_differences(lambda v: ours(n, v), lambda v: formula(n, v, 0), lambda v: formula(n, v, 1), x[n], got["d" + n],
                          want["d" + n][0], 0.4, 13)


# ------------------------------------------------------------------ calls --
def test_refusals():
    x, w, k = torch.zeros((2, 8), device=DEV), torch.zeros(8, device=DEV), key()
    for p in (-0.1, 1.0, 1.0 - 2.0 ** -18, float("nan")):
        for call in (lambda: learning.dropout(x, p, k), lambda: learning.layer_norm_residual(x, None, w, dropout=p, key=k)):
            with pytest.raises(ValueError):
                call()
    for bad in (dict(key=None), dict(key=k[:1]), dict(key=k.cpu()), dict(key=k, call=-1), dict(key=k, call=2 ** 32),
                dict(key=k, call=1.0), dict(key=k, call=True)):
        with pytest.raises(ValueError):
            learning.dropout(x, 0.5, **bad)
        with pytest.raises(ValueError):
            learning.layer_norm_residual(x, None, w, dropout=0.5, **bad)
    for bad in (k.int(), k.float(), (1, 2)):
        with pytest.raises(TypeError):
            learning.dropout(x, 0.5, bad)
    wide = torch.zeros((1, 1), device=DEV).expand(1, (1 << 24) + 1)
    for call in (lambda: learning.dropout(wide, 0.5, k), lambda: learning.layer_norm_residual(wide[:, :8193], None, wide[0, :8193]),
                 lambda: learning.layer_norm_residual(x, x[:1], w), lambda: learning.layer_norm_residual(x, None, w[:7]),
                 lambda: learning.layer_norm_residual(x, None, w, w[:7]), lambda: learning.layer_norm_residual(x, None, w, eps=-1.0),
                 lambda: learning.layer_norm_residual(x, None, w, eps=float("nan")),
                 lambda: learning.dropout(x[:, :1].expand(-1, 1)[:1].expand(1 << 31, 1), 0.5, k)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: learning.layer_norm_residual(x, None, None), lambda: learning.layer_norm_residual(x, None, w.bfloat16()),
                 lambda: learning.layer_norm_residual(x, x.bfloat16(), w), lambda: learning.layer_norm_residual(x, None, w, 1.0)):
        with pytest.raises(TypeError):
            call()


def test_a_key_advanced_too_early_is_seen_by_autograd():
    x, k = torch.randn(4, 8, device=DEV, requires_grad=True), key()
    y = learning.dropout(x, 0.5, k)
    k[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad

    x, w = torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, x)
        for call in (lambda: learning.dropout(d, 0.5, key()), lambda: learning.layer_norm_residual(d, None, w),
                     lambda: learning.layer_norm_residual(x, d, w),
                     lambda: learning.layer_norm_residual(x, None, w, forward_ad.make_dual(w, w))):
            with pytest.raises(NotImplementedError):
                call()


def test_saved_tensors_may_come_back_with_other_strides():
    x = norm_inputs(9, 200, torch.bfloat16, seed=14)
    want = norm_run(x, p=0.2, k=key())
    with torch.autograd.graph.save_on_cpu():
        got = norm_run(x, p=0.2, k=key())
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_captured_step_draws_new_masks():
    """A captured training step (norm with dropout, dropout, their gradients, the key's advance) gives on
    each replay what the eager step of that number gives."""
    x = norm_inputs(300, 264, torch.bfloat16, seed=15)
    k = key()
    leaf = [x[n].detach().requires_grad_(True) for n in ("x", "r", "w", "b")]

    def step(k):
        y, s = learning.layer_norm_residual(*leaf, dropout=0.1, key=k, call=0)
        z = learning.dropout(y, 0.3, k, call=1)
        return (z, s, *torch.autograd.grad([z, s], leaf, [x["dy"], x["ds"]]))

    eager = []
    for i in range(4):
        eager.append([t.detach().clone() for t in step(key(step=KEY[1] + i))])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(k)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(k)
        k[1] += 1
    for i in range(4):
        graph.replay()
        for a, b in zip(out, eager[i]):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
        learning.dropout(x["x"], 0.5, key())  # eager work between the replays
    assert not torch.equal(eager[0][0], eager[1][0])


def test_another_stream():
    x = norm_inputs(500, 264, torch.float32, seed=16)
    want = norm_run(x, p=0.1, k=key())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm_run(x, p=0.1, k=key())
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        assert torch.equal(got[n], want[n]), n
