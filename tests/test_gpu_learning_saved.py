"""The history model's operators under saved-tensor hooks that give tensors back with equal values and other
layouts: equal gradients."""
import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

from test_gpu_learning_calls import attention_inputs
from test_gpu_learning_delta import inputs
from test_gpu_learning_delta_gradients import run
from test_gpu_learning_norm import key, norm_inputs, norm_run
from test_learning_saved import spread, turned
from turbompc_amd import learning

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]
LAYOUTS = [spread, turned]


def given_back(layout, fn):
    with saved_tensors_hooks(lambda t: t, layout):
        return fn()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_delta_attention(layout, dtype):
    x = inputs(3, 40, (4, 2, 4, 1), 16, 24, dtype, lengths=[40, 0, 17])
    want = run(x)
    got = given_back(layout, lambda: run(x))
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_delta_attention_with_repeated_values():
    """A tensor of one value may come back as one element, expanded."""
    x = inputs(2, 40, (2, 2, 2, 2), 16, 24, torch.float32)
    x = dict(x, q=torch.ones_like(x["q"]), state=torch.ones_like(x["state"]))
    want = run(x)
    got = given_back(lambda t: t.flatten()[:1].reshape((1,) * t.dim()).expand(t.shape) if bool((t == 1).all()) else t, lambda: run(x))
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_layer_norm(layout, dtype):
    x = norm_inputs(9, 200, dtype, seed=14)
    want = norm_run(x, p=0.2, k=key())
    got = given_back(layout, lambda: norm_run(x, p=0.2, k=key()))
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_decay_attention(layout, dtype):
    q, k, v, g, state = attention_inputs(3, 40, 4, 2, 16, 24, dtype, seed=2)
    lengths = torch.tensor([40, 0, 17], dtype=torch.int32, device=DEV)

    def grads():
        leaf = [t.detach().requires_grad_(True) for t in (q, k, v, state)]
        o, s = learning.decay_attention(leaf[0], leaf[1], leaf[2], g, leaf[3], lengths)
        return torch.autograd.grad((o.float() ** 2).sum() + s.sum(), leaf)

    for a, b in zip(given_back(layout, grads), grads()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_rms_norm(layout, dtype):
    x = norm_inputs(9, 200, dtype, seed=15)

    def grads():
        leaf = [x[n].detach().requires_grad_(True) for n in ("x", "r", "w")]
        return torch.autograd.grad(learning.rms_norm_residual(*leaf), leaf, [x["dy"], x["ds"]])

    for a, b in zip(given_back(layout, grads), grads()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_gated_feed_forward(layout, dtype):
    gen = torch.Generator().manual_seed(16)
    data = [torch.randn(s, generator=gen).to(dtype).to(DEV) * 0.3 for s in ((9, 40), (72, 40), (72, 40), (24, 72), (9, 24))]

    def grads():
        leaf = [t.detach().requires_grad_(True) for t in data[:4]]
        return torch.autograd.grad(learning.gated_feed_forward(*leaf), leaf, data[4])

    for a, b in zip(given_back(layout, grads), grads()):
        assert torch.equal(a, b)
