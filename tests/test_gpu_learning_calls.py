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


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_of_a_long_history(dtype):
    """The stride of an axis of one entry is never used, however wide it is: the last step
    of one vehicle's log, with its rows 2^21 elements and more apart."""
    gen = torch.Generator().manual_seed(20)
    log = torch.randn((1, 9000, 256), generator=gen).to(dtype).to(DEV)
    wg, wu = (torch.randn((40, 256), generator=gen).to(dtype).to(DEV) / 16 for _ in range(2))
    wd, n = torch.randn((256, 40), generator=gen).to(dtype).to(DEV) / 8, torch.ones(256, dtype=dtype, device=DEV)
    ops = {"ff": lambda x: learning.gated_feed_forward(x, wg, wu, wd),
           "norm": lambda x: learning.rms_norm_residual(x, None, n)[0],
           "residual": lambda x: learning.rms_norm_residual(x * 2, x, n)[0]}
    row = log[:, -1]
    dy = log.flip(1)[:, 17]
    wide_dy = torch.randn((1, 9000, 256), generator=gen).to(dtype).to(DEV)[:, 3]
    assert row.stride(0) > 1 << 20 and wide_dy.stride(0) > 1 << 20
    for name, op in ops.items():
        for g in (dy, wide_dy):
            a = row.detach().requires_grad_(True)
            b = torch.empty(1, 256, dtype=dtype, device=DEV).copy_(row).requires_grad_(True)
            ya, yb = op(a), op(b)
            assert torch.equal(ya, yb), name
            ga, = torch.autograd.grad(ya, a, g)
            gb, = torch.autograd.grad(yb, b, torch.empty(1, 256, dtype=dtype, device=DEV).copy_(g))
            assert torch.equal(ga, gb), name


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_step_of_time_major_histories(dtype):
    B, H, d = 1100, 64, 128
    x = [torch.randn((1, B, H, d), generator=torch.Generator().manual_seed(s)).to(dtype).to(DEV) for s in range(4)]
    assert x[0].transpose(0, 1).stride(1) >= 1 << 23
    g = torch.full((H,), -0.5, device=DEV)

    def run(q, k, v, do):
        leaf = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o, s = learning.decay_attention(*leaf, g)
        return (o.detach(), s.detach(), *torch.autograd.grad(o, leaf, do))

    views = run(*(t.transpose(0, 1) for t in x))
    plain = run(*(torch.empty((B, 1, H, d), dtype=dtype, device=DEV).copy_(t.transpose(0, 1)) for t in x))
    for a, b in zip(views, plain):
        assert torch.equal(a, b)


def test_sizes_past_the_limits_are_value_errors():
    """Limits of the library are refused with the shape's name before anything is enqueued."""
    one = torch.zeros((1, 1, 1), device=DEV)
    heads = torch.zeros(32, device=DEV)
    B = (1 << 18) + 1  # 2^23 + 32 problems' heads
    q, state = one.expand(B, 32, 1), torch.zeros((B, 32, 1, 1), device=DEV)
    with pytest.raises(ValueError):
        learning.decay_attention_step(q, q, q, heads, state)
    with pytest.raises(ValueError):
        learning.decay_attention(*(t[:, None] for t in (q, q, q)), heads)
    w = torch.zeros((1, 1), device=DEV)
    with pytest.raises(ValueError):
        learning.gated_feed_forward(one[0].expand((1 << 30) + 1, 1), w, w, w)


def test_arguments_that_are_no_tensors_are_type_errors():
    x, w, wd = torch.zeros((2, 8), device=DEV), torch.zeros((4, 8), device=DEV), torch.zeros((8, 4), device=DEV)
    for args in ((None, w, w, wd), (x, None, w, wd), (x, w, None, wd), (x, w, w, None)):
        with pytest.raises(TypeError):
            learning.gated_feed_forward(*args)
    for args in ((None, None, wd[:, 0]), (x, 1.0, wd[:, 0]), (x, None, None)):
        with pytest.raises(TypeError):
            learning.rms_norm_residual(*args)
    q, g = torch.zeros((1, 2, 2, 8), device=DEV), torch.zeros(2, device=DEV)
    for args in ((None, q, q, g), (q, None, q, g), (q, q, None, g), (q, q, q, None), (q, q, q, g, 0.0)):
        with pytest.raises(TypeError):
            learning.decay_attention(*args)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_model_cast_after_it_was_made(dtype):
    """`to`, `bfloat16` and `float` cast the parameters; the decays stay float32, with their values."""
    model = learning.HistoryWeights(5, {"a": 2}, width=32, layers=2, heads=2, hidden=48,
                           dtype=torch.float32 if dtype == torch.bfloat16 else torch.bfloat16)
    decays = [b.log_decay.clone() for b in model.blocks]
    model = model.bfloat16() if dtype == torch.bfloat16 else model.to(dtype)
    assert all(p.dtype == dtype for p in model.parameters())
    assert all(b.log_decay.dtype == torch.float32 and torch.equal(b.log_decay, d) for b, d in zip(model.blocks, decays))
    history = torch.randn(3, 7, 5, device="cuda")
    w = model(history)["a"]
    w.sum().backward()
    assert bool(torch.isfinite(w).all()) and all(p.grad is not None for p in model.parameters())
    state = model.initial_state(3)
    model.step(history[:, 0], state)
    saved = model.state_dict()
    other = learning.HistoryWeights(5, {"a": 2}, width=32, layers=2, heads=2, hidden=48, dtype=dtype)
    other.load_state_dict(saved)
    assert torch.equal(other(history)["a"], model(history)["a"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_saved_tensors_may_come_back_with_other_strides(dtype):
    """Saved on the host between the passes, the views of a wider tensor return contiguous."""
    q, k, v, g, state = attention_inputs(2, 9, 2, 1, 16, 24, dtype)
    wide = torch.randn((30, 50), generator=torch.Generator().manual_seed(24)).to(dtype).to(DEV)
    w, wd = wide[:24, :16].contiguous() / 4, wide[:16, :24].contiguous() / 5

    def grads():
        x = wide[:, 3:19].detach().requires_grad_(True)
        p = torch.cat([q, k], 2).requires_grad_(True)
        y, s = learning.rms_norm_residual(learning.gated_feed_forward(x, w, w, wd), x, wd[:, 0])
        o, e = learning.decay_attention(p[:, :, :2], p[:, :, 2:], v, g, state)
        return torch.autograd.grad(y.sum() + s.sum() + o.sum() + e.sum(), [x, p])

    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_model_with_lengths_past_the_history():
    model = learning.HistoryWeights(5, {"a": 2}, width=32, layers=2, heads=2, hidden=48)
    history = torch.randn(4, 11, 5, device=DEV)
    with torch.no_grad():
        got = model(history, torch.tensor([11, 12, 500, -3], dtype=torch.int32, device=DEV))["a"]
        want = model(history, torch.tensor([11, 11, 11, 0], dtype=torch.int32, device=DEV))["a"]
    assert torch.equal(got, want)
