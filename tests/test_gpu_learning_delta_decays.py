"""log_decay's gradient where decays are strong (turbompc_amd.learning.delta_attention): the gradient carries the
decay as a factor, and its error is to be a few last bits of itself, not of what the step has in its outputs.

Judged in the norm of each head against |dg| alone, with the limit that the reference has for this gradient: six
products in a row of sums of n = T + dk + dv + 64 rounded terms, sqrt(n) units of 2^-24 each, eight
times that.  What it is summed up from (w_t, z_t and the ends' products of states) is of the gradients' own
size where decays are alike from step to step, and a larger end weighs less by its square."""
import pytest
import torch

import learning_reference_delta as ref
from test_gpu_learning_delta import DTYPES, inputs
from test_gpu_learning_delta_gradients import NAMES, run

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(x):
    do = x["do"] if x["do"] is not None else torch.zeros(x["g"].shape + x["v"].shape[-1:], dtype=x["q"].dtype)
    return ref.delta(*(x[n] for n in NAMES), x["lengths"], None, do, x["dstate"])


def assert_dg(x):
    value, _, limit, _ = reference(x)["dg"]
    got = run(x)["dg"]
    ref.assert_within("dg", got, (value, 0.0, limit, None), 2)
    return got, value


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("decay", [0.5, 3.0, 8.0, 15.0, 40.0])
@pytest.mark.parametrize("shape", [(2, 50, (2, 2, 2, 2), 32, 48), (1, 200, (4, 2, 2, 4), 64, 64), (1, 600, (2, 2, 1, 2), 20, 100),
                                   (1, 1100, (1, 1, 1, 1), 16, 16)], ids=lambda s: "x".join(map(str, s)).replace(" ", ""))
def test_decays_that_are_strong_throughout(shape, decay, dtype):
    """With and without a first state and a gradient of the last one; 1100 steps are cut into runs."""
    x = inputs(*shape, dtype, seed=int(decay) + shape[1])
    gen = torch.Generator().manual_seed(1)
    x["g"] = (-decay * torch.exp(0.3 * torch.randn(x["g"].shape, generator=gen))).to(DEV)
    for change in ({}, dict(dstate=None), dict(state=None), dict(state=None, dstate=None), dict(do=None)):
        assert_dg(dict(x, **change))


@pytest.mark.parametrize("dtype", DTYPES)
def test_ragged_histories_and_heads_of_different_decays(dtype):
    x = inputs(6, 300, (4, 4, 4, 4), 32, 32, dtype, seed=5, lengths=[300, 1, 33, 256, 257, 0])
    gen = torch.Generator().manual_seed(2)
    x["g"] = (-torch.tensor([0.05, 2.0, 9.0, 30.0]) * torch.exp(0.3 * torch.randn(x["g"].shape, generator=gen))).to(DEV)
    assert_dg(x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_zero_where_the_decay_is(dtype):
    """Below 2^-126 among ordinary steps, and in whole heads."""
    x = inputs(2, 150, (2, 2, 2, 2), 32, 32, dtype, seed=6)
    gone = [-88.0, -104.0, -1e4, -1e5, -1e30, -float("inf")]
    for i, g in enumerate(gone):
        x["g"][0, 20 * i + 3, 0] = g
        x["g"][1, 20 * i + 16, 1] = g
    got, _ = assert_dg(x)
    for i in range(len(gone)):
        assert got[0, 20 * i + 3, 0] == 0 and got[1, 20 * i + 16, 1] == 0
    x["g"][:, :, 1] = -200.0
    got, _ = assert_dg(x)
    assert not bool(got[:, :, 1].any()) and bool(got[:, :, 0].any())
