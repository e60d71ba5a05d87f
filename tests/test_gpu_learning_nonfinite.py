"""Infinities, NaN and huge values at one step of a history (turbompc_amd.learning): they reach
what the recurrence lets them reach, and no earlier step, other problem or other head."""
import pytest
import torch

import learning_reference as ref
from test_gpu_learning_attention import bounds, inputs, run
from turbompc_amd import learning

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
SHAPES = [(2, 150, 2, 1, 16, 24), (1, 150, 2, 2, 128, 128), (1, 101, 4, 2, 64, 128), (1, 75, 1, 1, 127, 33),
          (1, 1100, 1, 1, 32, 32)]


def reference(x, lengths=None):
    return ref.attention(x["q"], x["k"], x["v"], x["g"], x["state"], lengths, None, x["do"], x["dstate"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_non_finite_values_spoil_what_depends_on_them(shape, what, dtype):
    x = inputs(*shape, dtype, seed=21)
    T = shape[1]
    for at, value in ((T // 2, float("nan")), (T - 7, float("inf")), (3, float("-inf"))):
        bad = dict(x, **{what: x[what].clone()})
        bad[what][0, at, 0, 5] = value
        got = run(bad)
        for k, (v, tol) in bounds(bad, reference(bad), dtype).items():
            there = torch.isfinite(v)
            assert torch.equal(torch.isfinite(got[k]).cpu(), there), (k, at, value)
            over = (ref.cpu64(got[k]) - v).abs()[there] - (tol[there] + ref.TINY)
            assert float(over.max()) <= 0.0, (k, at, value, float(over.max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [1e30, -3e38])
def test_huge_values_leave_the_earlier_steps(value, dtype):
    """Products that overflow between a step and a later one belong to no output."""
    x = inputs(2, 90, 2, 1, 32, 48, dtype, seed=22)
    for at in (10, 64, 77):
        bad = {k: t.clone() if torch.is_tensor(t) else t for k, t in x.items()}
        for k in ("q", "k", "v"):
            bad[k][1, at] = value
        o, s = learning.decay_attention(bad["q"], bad["k"], bad["v"], x["g"], x["state"])
        cut = {k: x[k][:, :at] if k in ("q", "k", "v", "do") else x[k] for k in x}
        v, tol = bounds(cut, reference(cut), dtype)["o"]
        ref.assert_within("o", o[:, :at], v, tol)
        clean, _ = learning.decay_attention(x["q"][:1], x["k"][:1], x["v"][:1], x["g"], x["state"][:1])
        assert torch.equal(o[:1], clean)


def test_the_steps_after_a_spoiled_chunk_are_whole_again():
    """A strong decay (a factor of 2^-8 a step) forgets a huge value; lengths end inside its chunk."""
    x = inputs(3, 200, 1, 1, 16, 16, torch.float32, seed=23, g=-8 * 0.6931472)
    x["v"][:, 5] = 1e25
    lengths = torch.tensor([200, 6, 20], dtype=torch.int32, device="cuda")
    got = run(x, lengths)
    for k, (v, tol) in bounds(x, reference(x, lengths), torch.float32).items():
        ref.assert_within(k, got[k], v, tol)


@pytest.mark.parametrize("value", [0.5, float("inf")])
def test_a_state_given_and_returned_in_one_buffer(value):
    """A C caller may let state_out be state_in, whether or not a run has to be made again."""
    from turbompc_amd import _lib
    from turbompc_amd.learning import ops

    x = inputs(2, 100, 2, 1, 32, 48, torch.float32, seed=25)
    x["v"][1, 60, 0, 7] = value
    with torch.no_grad():
        want_o, want_s = learning.decay_attention(x["q"], x["k"], x["v"], x["g"], x["state"])
    state, o = x["state"].clone(), torch.empty_like(want_o)
    a = ops._attention_args(x["q"], x["k"], x["v"], x["g"], None, state, 32 ** -0.5)
    _lib.check("forward", _lib.load().tmpc_decay_attention_forward_f32(
        torch.cuda.current_stream().cuda_stream, a, o.data_ptr(), state.data_ptr(), None, 0))
    for got, want in ((o, want_o), (state, want_s)):
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        assert torch.equal(torch.isnan(got), torch.isnan(want))
