"""What a caller of the history model's operators may count on beside the values: limits,
views, torch's autograd rules."""
import pytest
import torch
from torch.autograd import forward_ad

from turbompc_amd import learning

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]


def test_histories_past_the_step_limit_are_refused():
    q = torch.zeros((1, 1, 1, 1), device=DEV)
    g = torch.zeros(1, device=DEV)
    for T in (2 ** 30 + 1, 2 ** 31):
        x = q.expand(1, T, 1, 1)  # no memory behind it
        with pytest.raises(ValueError):
            learning.decay_attention(x, x, x, g)


def attention_inputs(B, T, H, Hk, dk, dv, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s, dt=dtype: torch.randn(s, generator=gen).to(dt).to(DEV)  # noqa: E731
    g = torch.log1p(-torch.exp2(-torch.linspace(1, 6, H))).to(DEV)
    return r(B, T, H, dk), r(B, T, Hk, dk), r(B, T, Hk, dv), g, r(B, H, dk, dv, dt=torch.float32)


def test_a_step_on_a_saved_state_is_seen_by_autograd():
    """The backward pass reads the state that the forward call was given: overwritten in place
    before it, it is an error as with any in-place operation."""
    q, k, v, g, state = attention_inputs(2, 9, 2, 1, 16, 24, torch.float32)
    q.requires_grad_(True)
    o, s = learning.decay_attention(q, k, v, g, state)
    before = state._version
    with torch.no_grad():
        learning.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    o, s = learning.decay_attention(q, k, v, g, state.clone())  # another tensor's step is none of its business
    with torch.no_grad():
        learning.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state)
    o.sum().backward()
    assert bool(torch.isfinite(q.grad).all())


def test_a_step_in_inference_mode():
    q, k, v, g, state = attention_inputs(2, 1, 2, 1, 16, 24, torch.float32)
    want = state.clone()
    o = learning.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, want)
    with torch.inference_mode():
        inside = state.clone()
        for s in (state, inside):
            assert torch.equal(learning.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s), o)
            assert torch.equal(s, want)


def test_forward_mode_derivatives_are_refused():
    """A tangent is never dropped: there is no forward-mode rule, so a dual input is an error."""
    q, k, v, g, state = attention_inputs(2, 3, 2, 1, 8, 8, torch.float32)
    x, w, wd, n = torch.randn(4, 8, device=DEV), torch.randn(6, 8, device=DEV), torch.randn(8, 6, device=DEV), torch.ones(8, device=DEV)
    calls = {
        "attention": (learning.decay_attention, [q, k, v, g, state], (0, 1, 2, 3, 4)),
        "step": (learning.decay_attention_step, [q[:, 0], k[:, 0], v[:, 0], g, state], (0, 1, 2, 3, 4)),
        "feed_forward": (learning.gated_feed_forward, [x, w, w, wd], (0, 1, 2, 3)),
        "norm": (learning.rms_norm_residual, [x, x, n], (0, 1, 2)),
    }
    for name, (fn, args, places) in calls.items():
        for i in places:
            for mode in (torch.enable_grad, torch.no_grad):
                with forward_ad.dual_level(), mode():
                    dual = list(args)
                    dual[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                    with pytest.raises(NotImplementedError):
                        fn(*dual)
        with forward_ad.dual_level():
            fn(*args)  # no tangent among them: as anywhere else
