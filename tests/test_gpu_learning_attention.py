"""Decay attention (turbompc_amd.learning) against the step-by-step recurrence in 64 bits."""
import pytest
import torch

import learning_reference as ref
from turbompc_amd import learning

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]


def inputs(B, T, H, Hk, dk, dv, dtype, seed=0, state=True, g=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s, dt=dtype: torch.randn(s, generator=gen).to(dt).to(DEV)  # noqa: E731
    x = dict(q=r(B, T, H, dk), k=r(B, T, Hk, dk), v=r(B, T, Hk, dv), do=r(B, T, H, dv),
             state=r(B, H, dk, dv, dt=torch.float32) if state else None, dstate=r(B, H, dk, dv, dt=torch.float32))
    e = torch.linspace(1, 6, H)
    x["g"] = (torch.log1p(-torch.exp2(-e)) if g is None else torch.full((H,), g)).float().to(DEV)
    return x


def run(x, lengths=None, scale=None):
    """All outputs and gradients of one call."""
    leaf = {k: x[k].detach().requires_grad_(True) for k in ("q", "k", "v", "state") if x[k] is not None}
    o, s = learning.decay_attention(leaf["q"], leaf["k"], leaf["v"], x["g"], leaf.get("state"), lengths, scale)
    grads = torch.autograd.grad((o, s), list(leaf.values()), (x["do"], x["dstate"]))
    out = {"o": o.detach(), "state": s.detach()}
    out.update({"d" + k: t for k, t in zip(leaf, grads)})
    return out


def bounds(x, want, dtype):
    """The recurrence's values with the bounds of the chunked form: roundings of the scores,
    of the state as an operand and of the result (bf16), and fp32 sums of T and of the widths."""
    T, dk, dv, H = x["q"].shape[1], x["q"].shape[3], x["v"].shape[3], x["q"].shape[2]
    c = (T + dk + dv + H + 64) * 2 * ref.F32
    e = ref.unit(dtype) if dtype == torch.bfloat16 else 0.0
    low = {"state", "dstate"}  # fp32 results: no rounded operand enters
    return {k: (v, (c + (0 if k in low else 2 * e)) * m + (0 if k in low else ref.unit(dtype)) * v.abs())
            for k, (v, m) in want.items()}


def check(x, got, dtype, lengths=None, scale=None):
    want = ref.attention(x["q"], x["k"], x["v"], x["g"], x["state"], lengths, scale, x["do"], x["dstate"])
    for k, (v, tol) in bounds(x, want, dtype).items():
        if k in got:
            ref.assert_within(k, got[k], v, tol)


SHAPES = [  # B, T, H, Hk, dk, dv
    (2, 1, 2, 2, 16, 16), (1, 2, 1, 1, 1, 1), (2, 31, 2, 1, 33, 57), (1, 32, 3, 3, 32, 32), (2, 33, 4, 2, 64, 48),
    (1, 64, 2, 2, 64, 64), (2, 65, 2, 2, 128, 64), (1, 130, 2, 1, 20, 128), (1, 200, 1, 1, 127, 127),
    (3, 97, 6, 2, 48, 80),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(shape, dtype):
    x = inputs(*shape, dtype, seed=sum(shape))
    check(x, run(x), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("state", [False, True])
def test_ragged_lengths(state, dtype):
    x = inputs(7, 70, 4, 2, 24, 40, dtype, seed=3, state=state)
    lengths = torch.tensor([0, 1, 70, 33, 64, 500, -4], dtype=torch.int32, device=DEV)  # clamped to 0..70
    got = run(x, lengths)
    check(x, got, dtype, lengths)
    for k in ("o", "dq", "dk", "dv"):
        assert not got[k][0].any() and not got[k][1, 1:].any() and not got[k][6].any(), k
    start = x["state"] if state else torch.zeros_like(got["state"])
    assert torch.equal(got["state"][0], start[0])
    if state:
        assert torch.equal(got["dstate"][0], x["dstate"][0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_places_are_not_read(dtype):
    x = inputs(4, 70, 2, 1, 32, 64, dtype, seed=4)
    lengths = torch.tensor([0, 5, 64, 66], dtype=torch.int32, device=DEV)
    clean = run(x, lengths)
    bad = dict(x)
    past = torch.arange(70, device=DEV)[None] >= lengths[:, None]
    for k, v in (("q", float("nan")), ("k", float("inf")), ("v", float("-inf")), ("do", float("nan"))):
        bad[k] = torch.where(past[..., None, None], torch.full_like(x[k], v), x[k])
    for k, t in run(bad, lengths).items():
        assert torch.equal(t, clean[k]), k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("g", [0.0, -1e-4, -3.0, -200.0, float("-inf")])
def test_decays(g, dtype):
    x = inputs(1, 140, 1, 1, 16, 16, dtype, seed=5, g=g)
    check(x, run(x), dtype)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.25])
def test_scale(scale):
    x = inputs(1, 40, 2, 2, 16, 16, torch.float32, seed=6)
    check(x, run(x, scale=scale), torch.float32, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_inputs(dtype):
    """Views of one projection, rows with a step, expanded gradients: as contiguous copies."""
    B, T, H, d = 2, 67, 4, 24
    gen = torch.Generator().manual_seed(7)
    big = torch.randn((B, T, 3 * H, d + 1), generator=gen).to(dtype).to(DEV)
    x = inputs(B, T, H, H, d, d, dtype, seed=8)
    views = dict(x, q=big[:, :, :H, 1:], k=big[:, :, H:2 * H, 1:], v=big.transpose(1, 2)[:, 2 * H:, :, :d].transpose(1, 2),
                 do=torch.ones((), dtype=dtype, device=DEV).expand(B, T, H, d))
    copies = {k: (t.contiguous() if t is not None else None) for k, t in views.items()}
    assert not views["q"].is_contiguous()
    a, b = run(views), run(copies)
    for k in a:
        assert torch.equal(a[k], b[k]), k
    stepped = dict(x, q=torch.randn((B, T, H, 2 * d), generator=gen).to(dtype).to(DEV)[..., ::2])
    a, b = run(stepped), run(dict(stepped, q=stepped["q"].contiguous()))
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("dtype", DTYPES)
def test_continued_history_is_the_whole_one(dtype):
    """Two calls, the second from the first one's state; a long history over few heads."""
    T, cut = 3000, 1237
    x = inputs(1, T, 2, 1, 64, 32, dtype, seed=9)
    whole, s = learning.decay_attention(x["q"], x["k"], x["v"], x["g"], x["state"])
    o1, s1 = learning.decay_attention(x["q"][:, :cut], x["k"][:, :cut], x["v"][:, :cut], x["g"], x["state"])
    o2, s2 = learning.decay_attention(x["q"][:, cut:], x["k"][:, cut:], x["v"][:, cut:], x["g"], s1)
    want = ref.attention(x["q"], x["k"], x["v"], x["g"], x["state"])
    for k, got in (("o", whole), ("o", torch.cat([o1, o2], 1)), ("state", s), ("state", s2)):
        v, m = want[k]
        # the decays leave about 2^6 steps in a sum, so that many terms of fp32 rounding
        tol = (1200 * ref.F32 + (2 * ref.unit(dtype) if dtype == torch.bfloat16 and k == "o" else 0)) * m
        ref.assert_within(k, got, v, tol + (ref.unit(dtype) if k == "o" else 0) * v.abs())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [700, 4100])
def test_long_history_gradients(T, dtype):
    x = inputs(1, T, 2, 1, 32, 48, dtype, seed=10)
    lengths = torch.tensor([T - 5], dtype=torch.int32, device=DEV)
    check(x, run(x, lengths), dtype, lengths)


def test_equal_inputs_give_equal_bits():
    x = inputs(3, 300, 4, 1, 64, 64, torch.bfloat16, seed=11)
    a, b = run(x), run(x)
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_gradients_against_differences():
    """The operator is linear in each of q, k (with q, v fixed), v and the state: a central
    difference of any width has no truncation error, only the outputs' rounding."""
    x = inputs(2, 50, 4, 2, 24, 40, torch.float32, seed=12)
    got = run(x)

    def loss(y):
        o, s = learning.decay_attention(y["q"], y["k"], y["v"], x["g"], y["state"])
        return float((o.double() * x["do"].double()).sum() + (s.double() * x["dstate"].double()).sum())

    mags = ref.attention(x["q"], x["k"], x["v"], x["g"], x["state"])
    size = float((mags["o"][1] * ref.cpu64(x["do"]).abs()).sum() + (mags["state"][1] * ref.cpu64(x["dstate"]).abs()).sum())
    for k in ("q", "k", "v", "state"):
        d = torch.randn(x[k].shape, generator=torch.Generator().manual_seed(13)).to(DEV)
        diff = (loss(dict(x, **{k: x[k] + d})) - loss(dict(x, **{k: x[k] - d}))) / 2
        exact = float((got["d" + k].double() * d.double()).sum())
        assert abs(diff - exact) <= 200 * 2 * ref.F32 * 3 * size, (k, diff, exact)


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_past_32_bits(dtype):
    """An output of more than 2^31 elements: its last steps are those of a short history
    (the decay of 1/2 a step leaves nothing older than 200 steps in fp32)."""
    T, H, dv = 2 ** 31 // (16 * 128) + 1001, 16, 128
    gen = torch.Generator(device=DEV).manual_seed(14)
    r = lambda *s: torch.randn(s, generator=gen, device=DEV, dtype=dtype)  # noqa: E731
    q, k, v = r(1, T, 1, 16).expand(1, T, H, 16), r(1, T, 1, 16), r(1, T, 1, dv)
    g = torch.full((H,), -0.6931472, device=DEV)
    with torch.no_grad():
        o, s = learning.decay_attention(q, k, v, g)
        o2, s2 = learning.decay_attention(q[:, -256:], k[:, -256:], v[:, -256:], g)
    assert o.numel() > 2 ** 31
    e = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18
    scale = float(o2.abs().max())
    assert float((o[:, -40:].float() - o2[:, -40:].float()).abs().max()) <= e * scale
    assert float((s - s2).abs().max()) <= 2.0 ** -18 * float(s2.abs().max())
    del o, q, k, v
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 4, 2, 16, 16), (5, 2, 2, 33, 57), (2, 3, 1, 128, 128), (1, 1, 1, 1, 1),
                                   (300, 2, 1, 64, 20)])
def test_step(shape, dtype):
    B, H, Hk, dk, dv = shape
    x = inputs(B, 1, H, Hk, dk, dv, dtype, seed=15)
    want = bounds(x, ref.attention(x["q"], x["k"], x["v"], x["g"], x["state"]), dtype)
    s = x["state"].clone()
    o = learning.decay_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["g"], s)
    ref.assert_within("o", o, want["o"][0][:, 0], want["o"][1][:, 0])
    ref.assert_within("state", s, *want["state"])


def test_steps_walk_the_history_and_idle_problems_stay():
    x = inputs(6, 40, 4, 2, 24, 32, torch.float32, seed=16)
    lengths = torch.tensor([40, 0, 1, 20, 39, 7], dtype=torch.int32, device=DEV)
    want = bounds(x, ref.attention(x["q"], x["k"], x["v"], x["g"], x["state"], lengths), torch.float32)
    s = x["state"].clone()
    os = []
    for t in range(40):
        on = lengths > t
        q, k, v = (torch.where(on[:, None, None], x[n][:, t], float("nan")) for n in ("q", "k", "v"))
        os.append(learning.decay_attention_step(q, k, v, x["g"], s, active=on))
    ref.assert_within("o", torch.stack(os, 1), *want["o"])
    ref.assert_within("state", s, *want["state"])
    assert torch.equal(s[1], x["state"][1])


def test_other_stream_and_graph():
    x = inputs(2, 150, 2, 1, 32, 32, torch.bfloat16, seed=17)
    want = run(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x)
    torch.cuda.current_stream().wait_stream(side)
    for k in want:
        assert torch.equal(got[k], want[k]), k
    # one control period in a graph: the state moves on with every replay
    step = [x[n][:, 0].clone() for n in ("q", "k", "v")]
    s_eager, s_graph = x["state"].clone(), x["state"].clone()
    learning.decay_attention_step(*step, x["g"], x["state"].clone())  # the library is loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = learning.decay_attention_step(*step, x["g"], s_graph)
        of, sf = learning.decay_attention(x["q"], x["k"], x["v"], x["g"], x["state"])
    for i in range(4):
        for n, t in zip(("q", "k", "v"), step):
            t.copy_(x[n][:, i])
        graph.replay()
        torch.cuda.synchronize()
        oe = learning.decay_attention_step(*step, x["g"], s_eager)
        assert torch.equal(o, oe) and torch.equal(s_graph, s_eager)
        assert torch.equal(of, want["o"]) and torch.equal(sf, want["state"])


def test_empty_batches_and_histories():
    for B, T in ((0, 5), (2, 0), (0, 0)):
        x = inputs(B, T, 2, 1, 8, 8, torch.float32)
        got = run(x)
        assert got["o"].shape == (B, T, 2, 8)
        assert torch.equal(got["state"], x["state"]) and torch.equal(got["dstate"], x["dstate"])


def test_refusals():
    x = inputs(2, 5, 4, 2, 8, 8, torch.float32)
    call = lambda **kw: learning.decay_attention(**{**dict(  # noqa: E731
        q=x["q"], k=x["k"], v=x["v"], log_decay=x["g"], state=x["state"]), **kw})
    call()
    for err, kw in [
        (TypeError, dict(q=x["q"].double())), (TypeError, dict(k=x["k"].bfloat16())), (TypeError, dict(q=None)),
        (TypeError, dict(log_decay=x["g"].double())), (TypeError, dict(state=x["state"].bfloat16())),
        (TypeError, dict(lengths=torch.tensor([1, 2], device=DEV))),
        (ValueError, dict(q=x["q"].cpu())), (ValueError, dict(v=x["v"].cpu())), (ValueError, dict(q=x["q"][:, 0])),
        (ValueError, dict(k=x["k"][:, :3])), (ValueError, dict(v=x["v"][:, :, :1])),
        (ValueError, dict(q=x["q"][:, :, :3])), (ValueError, dict(log_decay=x["g"][:2])),
        (ValueError, dict(state=x["state"][:, :2])), (ValueError, dict(lengths=torch.ones(3, dtype=torch.int32, device=DEV))),
        (ValueError, dict(log_decay=x["g"].clone().requires_grad_(True))),
        (ValueError, dict(q=torch.zeros(2, 5, 4, 129, device=DEV), k=torch.zeros(2, 5, 2, 129, device=DEV), state=None)),
    ]:
        with pytest.raises(err):
            call(**kw)
    q, k, v = x["q"][:, 0], x["k"][:, 0], x["v"][:, 0]
    for err, kw in [(ValueError, dict(state=x["state"].transpose(2, 3))), (TypeError, dict(active=torch.ones(2, device=DEV))),
                    (ValueError, dict(q=q.clone().requires_grad_(True))), (ValueError, dict(q=x["q"]))]:
        with pytest.raises(err):
            learning.decay_attention_step(**{**dict(q=q, k=k, v=v, log_decay=x["g"], state=x["state"]), **kw})


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [6, 130])
def test_shared_heads_of_small_and_large_batches(B, dtype):
    """Key/value heads shared by four: the gradients are sums over a group's heads."""
    x = inputs(B, 70, 8, 2, 16, 24, dtype, seed=18)
    lengths = torch.arange(B, dtype=torch.int32, device=DEV) % 72
    check(x, run(x, lengths), dtype, lengths)
