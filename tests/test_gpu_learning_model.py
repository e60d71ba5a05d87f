"""The history model and its example: trained through the differentiable solve, and run row
by row as a control loop runs it."""
import sys
from pathlib import Path

import pytest
import torch

from turbompc_amd.learning import HistoryWeights

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_example_learns_and_runs_row_by_row(dtype):
    import learned_weights

    losses, model, history, lengths = learned_weights.run(B=48, steps=25, width=32, dtype=dtype, say=lambda s: None)
    assert all(torch.isfinite(torch.tensor(losses)))
    assert min(losses[-5:]) < 0.7 * losses[0], losses
    with torch.no_grad():
        whole = model(history, lengths)
    looped = learned_weights.control_loop(model, history, lengths)
    for k in whole:
        # the two forms round differently in every layer; bf16 has 8 bits
        tol = 1e-4 if dtype == torch.float32 else 2.0 ** -4
        assert float((whole[k] - looped[k]).abs().max()) <= tol * float(whole[k].abs().max()), k


def test_model_ignores_rows_past_a_history():
    model = HistoryWeights(5, {"a": 2, "b": 3}, width=32, layers=2, heads=2, hidden=48)
    history = torch.randn(6, 11, 5, device="cuda")
    lengths = torch.tensor([11, 0, 1, 4, 10, 7], dtype=torch.int32, device="cuda")
    want = model(history, lengths)
    past = torch.arange(11, device="cuda") >= lengths[:, None]
    got = model(torch.where(past[..., None], float("nan"), history), lengths)
    for k in want:
        assert torch.equal(got[k], want[k]) and bool((want[k] > 0).all()), k
    grads = torch.autograd.grad(sum(w.sum() for w in got.values()), list(model.parameters()))
    assert all(bool(torch.isfinite(g).all()) for g in grads)


def test_model_refuses_a_width_its_heads_do_not_divide():
    with pytest.raises(ValueError):
        HistoryWeights(5, {"a": 2}, width=30, heads=4)
