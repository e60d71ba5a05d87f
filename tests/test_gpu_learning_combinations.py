"""Decay attention (turbompc_amd.learning) where several of its cases meet: histories cut into runs
with every head width, ragged batches among them, weak decays over many chunks, 128 x 128 heads."""
import pytest
import torch

from test_gpu_learning_attention import DTYPES, check, inputs, run

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 31, 64, 130])
def test_128_wide_heads(T, dtype):
    """Whole pieces: the form that shares its scores out."""
    x = inputs(2, T, 2, 1, 128, 128, dtype, seed=41)
    lengths = torch.tensor([T, T // 3], dtype=torch.int32, device=DEV)
    check(x, run(x), dtype)
    check(x, run(x, lengths), dtype, lengths)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("widths", [(128, 128), (33, 57), (64, 32), (32, 128), (127, 20)], ids=str)
def test_runs_of_every_width(widths, dtype):
    """1100 steps of two heads are cut into runs of four or more chunks."""
    x = inputs(1, 1100, 2, 1, *widths, dtype, seed=42)
    check(x, run(x), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("widths", [(64, 32), (128, 128), (17, 40)], ids=str)
def test_runs_of_ragged_batches(widths, state, dtype):
    """Whole runs past a history's end, ends inside a run and on its edge, histories of nothing."""
    T = 1100
    x = inputs(5, T, 2, 2, *widths, dtype, seed=43, state=state)
    lengths = torch.tensor([0, 40, T - 5, 512, 1], dtype=torch.int32, device=DEV)
    got = run(x, lengths)
    check(x, got, dtype, lengths)
    for k in ("o", "dq", "dk", "dv"):
        for b, n in enumerate(lengths.tolist()):
            assert not got[k][b, n:].any(), (k, b)
    if state:
        assert torch.equal(got["state"][0], x["state"][0]) and torch.equal(got["dstate"][0], x["dstate"][0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("g", [0.0, -1e-4, -0.01])
@pytest.mark.parametrize("heads", [1, 260])
def test_weak_decays_over_many_chunks(heads, g, dtype):
    """2000 steps that hardly fade, in runs and (260 heads) whole."""
    T = 2000 if heads == 1 else 700
    x = inputs(1, T, heads, heads, 16, 16, dtype, seed=44, g=g)
    check(x, run(x), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shared_heads_in_runs(dtype):
    x = inputs(2, 1300, 4, 1, 64, 48, dtype, seed=45)
    lengths = torch.tensor([1300, 700], dtype=torch.int32, device=DEV)
    check(x, run(x, lengths), dtype, lengths)
