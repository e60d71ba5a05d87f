"""What the backward passes of the history model's operators hand to their kernels where a saved-tensor hook has
given a tensor back with equal values and another layout: the kernels' view of the memory has the values.  On
the CPU, the calls being recorded and not made."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from turbompc_amd.learning import delta_ops, norm_ops, ops

DTYPES = [torch.float32, torch.bfloat16]


def spread(t):
    """t's values, three elements apart."""
    wide = torch.full(t.shape + (3,), 7, dtype=t.dtype, device=t.device)
    wide[..., 1] = t
    return wide[..., 1]


def turned(t):
    """t's values with its axes in memory the other way round."""
    axes = tuple(range(t.dim()))[::-1]
    return t.permute(axes).contiguous().permute(axes)


def given_back(tensors, layout):
    return tuple(layout(t) if t is not None else None for t in tensors)


def at(address, shape, strides, dtype):
    """The values that a kernel reads from an address by these strides (elements)."""
    size = torch.empty((), dtype=dtype).element_size()
    n = 1 + sum((d - 1) * s for d, s in zip(shape, strides))
    raw = bytearray(ctypes.string_at(address, n * size))
    return torch.frombuffer(raw, dtype=dtype).as_strided(shape, strides).clone()


def rows_at(address, t):
    strides = torch.empty(t.shape).stride()
    return at(address, t.shape, strides, t.dtype)


@pytest.fixture
def calls(monkeypatch):
    """The operators' calls of the library, each read by the function that a test puts here."""
    readers = []

    def call(fn, device, *args):
        readers[0](fn, *args)

    for module in (ops, delta_ops, norm_ops):
        monkeypatch.setattr(module, "_call", call)
        monkeypatch.setattr(module, "_workspace", lambda *a: (0, None))
    return readers


def history(B, T, heads, d, dtype, seed):
    return torch.randn((B, T, heads, d), generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("layout", [spread, turned])
@pytest.mark.parametrize("dtype", DTYPES)
def test_delta_attention(calls, dtype, layout):
    B, T, H, dk, dv = 3, 5, 4, 8, 6
    gen = torch.Generator().manual_seed(1)
    saved = (history(B, T, 2, dk, dtype, 2), history(B, T, 4, dk, dtype, 3), history(B, T, 1, dv, dtype, 4),
             -torch.rand((B, T, H), generator=gen), torch.rand((B, T, H), generator=gen).to(dtype),
             torch.randn((B, H, dk, dv), generator=gen), torch.tensor([5, 2, 0], dtype=torch.int32))
    seen = []

    def read(fn, a, *rest):
        heads = lambda t, p, s: at(p, t.shape, (s[0], s[1], s[2], 1)[:t.dim()], t.dtype)  # noqa: E731
        q, k, v, g, beta, state, lengths = saved
        for t, p, s in ((q, a.q, a.q_stride), (k, a.k, a.k_stride), (v, a.v, a.v_stride), (g, a.log_decay, a.log_decay_stride),
                        (beta, a.beta, a.beta_stride)):
            assert torch.equal(heads(t, p, list(s)), t)
        assert torch.equal(rows_at(a.state_in, state), state) and torch.equal(rows_at(a.lengths, lengths), lengths)
        seen.append(fn)

    calls.append(read)
    ctx = SimpleNamespace(saved_tensors=given_back(saved, layout), scale=0.5, sfx="f32", needs_input_grad=(True,) * 9)
    with torch.no_grad():
        grads = delta_ops._DeltaAttention.backward(ctx, torch.zeros((B, T, H, dv), dtype=dtype), None)
    assert seen
    for g, t in zip(grads, saved[:6]):
        assert g.shape == t.shape and g.is_contiguous()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_and_dropout(calls, dtype):
    """All that is saved, the key's two words among it."""
    M, D = 5, 12
    gen = torch.Generator().manual_seed(5)
    x, r, dy = (torch.randn((M, D), generator=gen).to(dtype) for _ in range(3))
    w, stats, key = torch.randn(D, generator=gen).to(dtype), torch.rand((M, 2), generator=gen), torch.tensor([11, 12])
    seen = []

    def read(fn, *args):
        seen.append(fn)
        if "dropout" in fn:
            assert torch.equal(rows_at(args[5], key), key)
            return
        a, stats_at = args[0], args[7]
        assert torch.equal(at(a.x, (M, D), (a.ldx, 1), dtype), x) and torch.equal(at(a.residual, (M, D), (a.ldr, 1), dtype), r)
        assert torch.equal(rows_at(a.weight, w), w) and torch.equal(rows_at(stats_at, stats), stats)
        assert torch.equal(rows_at(a.key, key), key)

    calls.append(read)
    for layout in (spread, turned):
        saved = given_back((None, x, r, w, stats, key), layout)
        ctx = SimpleNamespace(saved_tensors=saved, args=(1e-5, 0.5, 0, "f32", True, True))
        with torch.no_grad():
            for g, t in zip(norm_ops._LayerNorm.backward(ctx, dy, None), (x, r, w, w)):
                assert g.shape == t.shape and g.is_contiguous()
            norm_ops._Dropout.backward(SimpleNamespace(saved_tensors=(layout(key),), args=(0.5, 0, "f32")), dy)
    assert len(seen) == 4


@pytest.mark.parametrize("layout", [spread, turned])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decay_attention(calls, dtype, layout):
    B, T, H, dk, dv = 3, 5, 4, 8, 6
    gen = torch.Generator().manual_seed(6)
    saved = (history(B, T, H, dk, dtype, 7), history(B, T, 2, dk, dtype, 8), history(B, T, 2, dv, dtype, 9),
             -torch.rand(H, generator=gen), torch.randn((B, H, dk, dv), generator=gen), torch.tensor([5, 2, 0], dtype=torch.int32))
    seen = []

    def read(fn, a, *rest):
        q, k, v, g, state, lengths = saved
        for t, p, s in ((q, a.q, a.q_stride), (k, a.k, a.k_stride), (v, a.v, a.v_stride)):
            assert torch.equal(at(p, t.shape, (*s, 1), dtype), t)
        for t, p in ((g, a.log_decay), (state, a.state_in), (lengths, a.lengths)):
            assert torch.equal(rows_at(p, t), t)
        seen.append(fn)

    calls.append(read)
    ctx = SimpleNamespace(saved_tensors=given_back(saved, layout), scale=0.5, sfx="f32", needs_input_grad=(True,) * 8)
    with torch.no_grad():
        grads = ops._DecayAttention.backward(ctx, torch.zeros((B, T, H, dv), dtype=dtype), None)
    assert seen
    for g, t in zip(grads[:3], saved):
        assert g.shape == t.shape and g.is_contiguous()


@pytest.mark.parametrize("layout", [spread, turned])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rms_norm(calls, dtype, layout):
    M, D = 5, 12
    gen = torch.Generator().manual_seed(10)
    s, dy = (torch.randn((M, D), generator=gen).to(dtype) for _ in range(2))
    w, rstd = torch.randn(D, generator=gen).to(dtype), torch.rand(M, generator=gen)
    seen = []

    def read(fn, dev, rows, width, dy_at, lddy, ds_at, ldds, s_at, lds, w_at, rstd_at, *rest):
        assert torch.equal(at(s_at, (M, D), (lds, 1), dtype), s)
        assert torch.equal(rows_at(w_at, w), w) and torch.equal(rows_at(rstd_at, rstd), rstd)
        seen.append(fn)

    calls.append(lambda fn, *args: read(fn, None, *args))
    ctx = SimpleNamespace(saved_tensors=given_back((s, w, rstd), layout), sfx="f32", has_residual=True)
    with torch.no_grad():
        dx, dr, dw, *_ = ops._RmsNorm.backward(ctx, dy, None)
    assert seen and dx.is_contiguous() and dx.shape == s.shape and dw.is_contiguous() and dr is dx


@pytest.mark.parametrize("layout", [spread, turned])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_feed_forward(calls, dtype, layout):
    M, D, F, out = 5, 12, 7, 6
    gen = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(s, generator=gen).to(dtype)  # noqa: E731
    x, w_gate, w_up, w_down = r(M, D), r(F, D), r(F, D), r(out, F)
    gate, up = torch.randn((M, F), generator=gen), torch.randn((M, F), generator=gen)
    seen = []

    def read(fn, a, gate_at, up_at, *rest):
        assert torch.equal(at(a.x, (M, D), (a.ldx, 1), dtype), x)
        for t, p in ((w_gate, a.w_gate), (w_up, a.w_up), (w_down, a.w_down), (gate, gate_at), (up, up_at)):
            assert torch.equal(rows_at(p, t), t)
        seen.append(fn)

    calls.append(read)
    ctx = SimpleNamespace(saved_tensors=given_back((x, w_gate, w_up, w_down, gate, up), layout), shape=x.shape, act=0, sfx="f32")
    with torch.no_grad():
        grads = ops._GatedFF.backward(ctx, r(M, out))
    assert seen
    for g, t in zip(grads, (x, w_gate, w_up, w_down)):
        assert g.shape == t.shape and g.is_contiguous()
