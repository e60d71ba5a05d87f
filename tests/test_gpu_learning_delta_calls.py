"""What a caller of the gated delta rule, the layer norm and dropout may count on beside the values:
refusals, torch's autograd rules, streams, graphs, and the history model that uses them together."""
import sys
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_learning_delta import inputs
from test_gpu_learning_delta_gradients import NAMES, run
from turbompc_amd import learning

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]


def args(x, **change):
    z = dict(x, **change)
    return [z[n] for n in NAMES]


def test_refusals():
    x = inputs(2, 5, (4, 2, 4, 1), 16, 24, torch.float32)
    H4 = torch.zeros(2, 5, 4, device=DEV)
    for change in (dict(k=x["k"][:, :4]), dict(k=x["k"][..., :8]), dict(v=x["v"][:1]), dict(g=x["g"][:, :4]), dict(g=x["g"][..., :3]),
                   dict(beta=x["beta"][..., :2]), dict(q=x["q"][:, 0]), dict(g=H4[0]), dict(state=x["state"][:1]),
                   dict(q=x["q"].cpu()), dict(g=x["g"].cpu()), dict(v=x["v"][..., :0]), dict(q=x["q"][:, :, :0]),
                   dict(k=torch.zeros(2, 5, 4, 129, device=DEV), q=torch.zeros(2, 5, 2, 129, device=DEV))):
        with pytest.raises(ValueError):
            learning.delta_attention(*args(x, **change))
    for change in (dict(q=None), dict(k=x["k"].bfloat16()), dict(g=x["g"].bfloat16()), dict(g=None), dict(beta=x["beta"].bfloat16()),
                   dict(state=x["state"].bfloat16()), dict(beta=0.5), dict(q=x["q"].half())):
        with pytest.raises(TypeError):
            learning.delta_attention(*args(x, **change))
    for lengths in (torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            learning.delta_attention(*args(x), lengths)
    with pytest.raises(TypeError):
        learning.delta_attention(*args(x), torch.zeros(2, dtype=torch.int64, device=DEV))
    one = [x[n][:, 0] for n in NAMES[:5]]
    for state in (x["state"].transpose(-1, -2), x["state"][:, :, ::2]):
        with pytest.raises(ValueError):
            learning.delta_attention_step(*one, state)
    with pytest.raises(TypeError):
        learning.delta_attention_step(*one, x["state"], active=torch.ones(2, device=DEV))
    with pytest.raises(ValueError):
        learning.delta_attention_step(*one, x["state"], active=torch.ones(3, dtype=torch.bool, device=DEV))
    one[0] = one[0].clone().requires_grad_(True)
    with pytest.raises(ValueError, match="gradient"):
        learning.delta_attention_step(*one, x["state"])


def test_sizes_past_the_limits_are_value_errors():
    for T in (2 ** 30 + 1, 2 ** 31):  # no memory behind them
        q, g = torch.zeros((1, 1, 1, 1), device=DEV).expand(1, T, 1, 1), torch.zeros((1, 1, 1), device=DEV).expand(1, T, 1)
        with pytest.raises(ValueError):
            learning.delta_attention(q, q, q, g, g)
    q, g = torch.zeros((1, 1, 1), device=DEV), torch.zeros((1, 1), device=DEV)
    B = (1 << 18) + 1
    with pytest.raises(ValueError):
        learning.delta_attention_step(q.expand(B, 1, 1), q.expand(B, 1, 1), q.expand(B, 1, 1), g.expand(B, 32), g.expand(B, 32),
                                      torch.zeros((B, 32, 1, 1), device=DEV))
    with pytest.raises(ValueError):
        learning.delta_attention(*(q.expand(1, 2, 1)[:, :, None] for _ in range(3)), g[..., None].expand(1, 2, 32769),
                                 g[..., None].expand(1, 2, 32769))


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_batches_and_histories(dtype):
    for B, T in ((0, 5), (2, 0)):
        x = inputs(B, T, (2, 2, 1, 2), 16, 24, dtype)
        got = run(x)
        assert got["o"].shape == (B, T, 2, 24)
        assert torch.equal(got["state"], x["state"]) and torch.equal(got["dstate"], x["dstate"])
        for n in ("q", "k", "v", "g", "beta"):
            assert got["d" + n].shape == x[n].shape


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_of_a_long_log_and_time_major_histories(dtype):
    """The stride of an axis of one entry is never used, however wide it is; steps too far apart are copied."""
    B, H, d = 1100, 64, 128
    gen = torch.Generator().manual_seed(3)
    t = [torch.randn((1, B, H, d), generator=gen).to(dtype).to(DEV) * 0.1 for _ in range(3)]
    gates = [-torch.rand((1, B, H), generator=gen).to(DEV), torch.rand((1, B, H), generator=gen).to(dtype).to(DEV)]
    views = [z.transpose(0, 1) for z in (*t, *gates)]
    assert views[0].stride(1) >= 1 << 23
    plain = [torch.empty(z.shape, dtype=z.dtype, device=DEV).copy_(z) for z in views]
    with torch.no_grad():
        for a, b in zip(learning.delta_attention(*views), learning.delta_attention(*plain)):
            assert torch.equal(a, b)
        del plain
        two = torch.zeros((2, 1, 4097 * 2048), dtype=dtype, device=DEV)[..., :16].unflatten(-1, (1, 16)).transpose(0, 1)
        g = torch.zeros((2, 1, 1 << 23), device=DEV)[..., :1].transpose(0, 1)
        assert two.stride(1) >= 1 << 23 and g.stride(1) >= 1 << 23
        o, s = learning.delta_attention(two + 1, two.add_(1), two, g, torch.ones((1, 2, 1), dtype=dtype, device=DEV))
        want = learning.delta_attention(*(z.contiguous() for z in (two, two, two, g)), torch.ones((1, 2, 1), dtype=dtype, device=DEV))
        assert torch.equal(o, want[0]) and torch.equal(s, want[1])


def test_forward_mode_derivatives_are_refused():
    x = inputs(2, 3, (2, 2, 2, 2), 8, 8, torch.float32)
    one = [x[n][:, 0] for n in NAMES[:5]] + [x["state"]]
    for fn, a in ((learning.delta_attention, args(x)), (learning.delta_attention_step, one)):
        for i in range(6):
            for mode in (torch.enable_grad, torch.no_grad):
                with forward_ad.dual_level(), mode():
                    dual = list(a)
                    dual[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
                    with pytest.raises(NotImplementedError):
                        fn(*dual)


def test_a_step_on_a_saved_state_is_seen_by_autograd():
    x = inputs(2, 9, (2, 2, 2, 2), 16, 24, torch.float32)
    q = x["q"].clone().requires_grad_(True)
    o, _ = learning.delta_attention(*args(x, q=q))
    before = x["state"]._version
    with torch.no_grad():
        learning.delta_attention_step(*(x[n][:, 0] for n in NAMES[:5]), x["state"])
    assert x["state"]._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    with torch.inference_mode():
        learning.delta_attention_step(*(x[n][:, 0] for n in NAMES[:5]), x["state"].clone())


@pytest.mark.parametrize("dtype", DTYPES)
def test_saved_tensors_may_come_back_with_other_strides(dtype):
    x = inputs(2, 40, (4, 2, 2, 4), 16, 24, dtype)
    proj = torch.cat([x["q"], x["k"]], 2)
    x = dict(x, q=proj[:, :, :2], k=proj[:, :, 2:], g=x["g"].permute(2, 1, 0).contiguous().permute(2, 1, 0))
    want = run(x)
    with torch.autograd.graph.save_on_cpu():
        got = run(x)
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_another_stream_and_two_calls_at_once():
    """Calls on two streams at the same time have workspaces of their own."""
    xs = [inputs(1, 1300, (2, 2, 2, 2), 64, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [run(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(xs[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for n in b:
            assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("T", [70, 1300])
def test_captured_training_step(T):
    """Forward and backward, captured and replayed, whole and in runs, between eager work."""
    x = inputs(2, T, (2, 1, 2, 2), 32, 48, torch.bfloat16, seed=4)
    want = run(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(x)
        graphs.append((graph, out))
    v = x["v"].clone()
    for i in range(3):
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for n in want:
                assert torch.equal(out[n], want[n]), n
        x["v"].zero_()  # the graphs read their inputs again
        graphs[0][0].replay()
        run(x)
        assert not torch.equal(graphs[0][1]["o"], want["o"])
        x["v"].copy_(v)


def test_captured_step_walks_on():
    x = inputs(3, 1, (2, 2, 1, 2), 32, 32, torch.bfloat16, seed=5)
    one = [x[n][:, 0] for n in NAMES[:5]]
    state, want = x["state"].clone(), x["state"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        learning.delta_attention_step(*one, state.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = learning.delta_attention_step(*one, state)
    for _ in range(4):
        graph.replay()
        w = learning.delta_attention_step(*one, want)
        assert torch.equal(o, w) and torch.equal(state, want)


# ------------------------------------------------------------------ model --
MODELS = [dict(memory="delta"), dict(norm="layer"), dict(memory="delta", norm="layer", dropout=0.1), dict(dropout=0.2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("options", MODELS, ids=lambda o: "-".join(map(str, o.values())))
def test_model_whole_and_row_by_row(options, dtype):
    torch.manual_seed(0)
    model = learning.HistoryWeights(5, {"a": 2, "b": 3}, width=48, layers=2, heads=4, kv_heads=2, hidden=72, dtype=dtype, **options)
    with torch.no_grad():
        model.w_heads.normal_()
    history = torch.randn(6, 40, 5, device=DEV)
    lengths = torch.tensor([40, 1, 17, 39, 32, 5], dtype=torch.int32, device=DEV)
    key = torch.tensor([7, 0], device=DEV)
    grads = []
    for step in (0, 1):
        w = model(history, lengths, key)
        grads.append(torch.autograd.grad(sum(v.sum() for v in w.values()), list(model.parameters())))
        key[1] += 1
    for g in grads[0]:
        assert bool(torch.isfinite(g).all()) and bool(g.any())
    same = all(torch.equal(a, b) for a, b in zip(*grads))
    assert same == (options.get("dropout", 0.0) == 0.0)
    model.eval()
    with torch.no_grad():
        whole = model(history, lengths)
        past = torch.arange(40, device=DEV) >= lengths[:, None]
        again = model(torch.where(past[..., None], float("nan"), history), lengths)
        state, last = model.initial_state(6), None
        for t in range(40):
            active = lengths > t
            w = model.step(history[:, t], state, active)
            last = w if last is None else {k: torch.where(active[:, None], w[k], last[k]) for k in w}
    for k in whole:
        assert torch.equal(whole[k], again[k])
        # the two forms round differently in every layer; bf16 has 8 bits
        tol = 1e-4 if dtype == torch.float32 else 2.0 ** -4
        assert float((whole[k] - last[k]).abs().max()) <= tol * float(whole[k].abs().max()), k


def test_example_runs_with_the_further_operators():
    import learned_weights

    losses, model, history, lengths = learned_weights.run(B=32, steps=4, width=32, say=lambda s: None, memory="delta", norm="layer",
                                                          dropout=0.1)
    assert all(torch.isfinite(torch.tensor(losses))) and not model.training
    looped = learned_weights.control_loop(model, history, lengths)
    assert all(bool(torch.isfinite(w).all()) for w in looped.values())


def test_model_training_step_captured():
    """A whole training step of the model with all of them in a graph: each replay's gradients are the
    eager step's of that number."""
    torch.manual_seed(1)
    model = learning.HistoryWeights(5, {"a": 2}, width=32, layers=2, heads=2, hidden=48, dtype=torch.bfloat16, memory="delta",
                                    norm="layer", dropout=0.1)
    with torch.no_grad():
        model.w_heads.normal_()
    history = torch.randn(4, 50, 5, device=DEV)
    params = list(model.parameters())
    key = torch.tensor([9, 0], device=DEV)

    def step(key):
        return torch.autograd.grad(model(history, None, key)["a"].sum(), params)

    want = []
    for i in range(3):
        want.append([g.clone() for g in step(torch.tensor([9, i], device=DEV))])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(key)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step(key)
        key[1] += 1
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(grads, want[i]):
            assert torch.equal(a, b)
