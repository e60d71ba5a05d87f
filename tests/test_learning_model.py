"""The history model's own arithmetic without a GPU: its operators are replaced by plain
torch forms, so that its indexing runs, bounds checked, on the CPU."""
import pytest
import torch

from turbompc_amd.learning import HistoryWeights, weights_model


def norm(x, residual, weight, eps=1e-6):
    s = x if residual is None else x + residual
    return s * torch.rsqrt((s * s).mean(-1, keepdim=True) + eps) * weight, s


def attention(q, k, v, log_decay, state=None, lengths=None, scale=None):
    B, T, H, d = q.shape
    k, v = (t.repeat_interleave(H // t.shape[2], dim=2) for t in (k, v))
    S = torch.zeros((B, H, d, v.shape[-1])) if state is None else state
    n = torch.full((B,), T) if lengths is None else lengths.clamp(0, T)
    o = torch.zeros((B, T, H, v.shape[-1]))
    for t in range(T):
        on = (n > t)[:, None, None]
        S = torch.where(on[..., None], torch.exp(log_decay)[:, None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :], S)
        o[:, t] = torch.where(on, d ** -0.5 * (q[:, t, :, None, :] @ S)[..., 0, :], 0.0)
    return o, S


def feed_forward(x, w_gate, w_up, w_down, activation="silu"):
    return (torch.nn.functional.silu(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(weights_model.ops, "rms_norm_residual", norm)
    monkeypatch.setattr(weights_model.ops, "decay_attention", attention)
    monkeypatch.setattr(weights_model.ops, "gated_feed_forward", feed_forward)
    torch.manual_seed(0)
    m = HistoryWeights(5, {"a": 2, "b": 3}, width=16, layers=2, heads=2, hidden=24, device="cpu")
    with torch.no_grad():
        m.w_heads.normal_()
    return m


def test_lengths_outside_the_history_are_clamped(model):
    history = torch.randn(6, 7, 5)
    got = model(history, torch.tensor([8, 500, 2 ** 31 - 1, 0, -4, 3], dtype=torch.int32))
    want = model(history, torch.tensor([7, 7, 7, 0, 0, 3], dtype=torch.int32))
    for k in want:
        assert torch.equal(got[k], want[k]), k
    for k, w in model(history).items():
        assert torch.equal(got[k][:3], w[:3]), k


@pytest.mark.parametrize("lengths", [None, torch.zeros(3, dtype=torch.int32)])
def test_histories_without_a_row_are_refused(model, lengths):
    with pytest.raises(ValueError):
        model(torch.zeros(3, 0, 5), lengths)


def test_a_cast_leaves_the_decays():
    m = HistoryWeights(5, {"a": 2}, width=16, layers=2, heads=2, device="cpu")
    decays = [b.log_decay.clone() for b in m.blocks]
    for cast in (lambda: m.bfloat16(), lambda: m.to(torch.float64), lambda: m.to("cpu", torch.float32)):
        assert cast() is m
        for b, d in zip(m.blocks, decays):
            assert b.log_decay.dtype == torch.float32 and torch.equal(b.log_decay, d)
            assert "log_decay" in dict(b.named_buffers())
