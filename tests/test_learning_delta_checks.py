"""The gated delta rule without a GPU: what the C entry points and the Python layer refuse before
anything is enqueued, the workspace queries, and the model's options."""
import ctypes

import pytest
import torch

from turbompc_amd import _lib, learning

SFX = ["f32", "bf16"]
X = ctypes.c_void_p(0x1000)  # never read: every call below returns before a launch


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def attention(**kw):
    a = dict(B=2, T=5, H=4, Hq=2, Hk=4, Hv=1, dk=16, dv=16)
    a.update(kw)
    return _lib.DeltaAttention(**a)


DATA = dict(q=X.value, k=X.value, v=X.value, beta=X.value, log_decay=X.value)


@pytest.mark.parametrize("sfx", SFX)
def test_refusals(lib, sfx):
    fwd, bwd, step = (getattr(lib, f"tmpc_delta_attention_{n}_{sfx}") for n in ("forward", "backward", "step"))
    st = (ctypes.c_int64 * 3)(1, 1, 1)
    back = lambda a, dos=st, ws=X, n=1 << 60: bwd(None, ctypes.byref(a), X, dos, None, X, X, X, X, X, X, ws, n)  # noqa: E731
    for bad in (dict(Hq=3), dict(Hk=3), dict(Hv=0), dict(H=0), dict(dk=0), dict(dk=129), dict(dv=129), dict(B=-1), dict(T=-1),
                dict(T=2 ** 30 + 1), dict(B=2 ** 30), dict(H=65536, Hq=1, Hk=1, Hv=1)):
        a = attention(**bad)
        assert fwd(None, ctypes.byref(a), X, X, X, 1 << 60) == 1, bad
        assert back(a) == 1, bad
        a.T = 1 if "T" not in bad else a.T
        assert step(None, ctypes.byref(a), None, X, X) == 1, bad
    assert fwd(None, None, X, X, X, 1 << 60) == 1
    wide = (ctypes.c_int64 * 3)(0, 1 << 23, 0)
    for name in ("q", "k", "v", "beta", "log_decay"):
        a = attention(**DATA, **{name + "_stride": wide})
        assert fwd(None, ctypes.byref(a), X, X, X, 1 << 60) == 1, name
        assert back(a) == 1, name
    assert back(attention(**DATA), wide) == 1
    for name in DATA:
        a = attention(**{**DATA, name: None})
        assert fwd(None, ctypes.byref(a), X, X, X, 1 << 60) == 2, name
        assert back(a) == 2, name
        a.T = 1
        assert step(None, ctypes.byref(a), None, X, X) == 2, name
    ok = attention(**DATA)
    assert fwd(None, ctypes.byref(ok), None, X, X, 1 << 60) == 2
    assert back(ok, None) == 2
    assert step(None, ctypes.byref(ok), None, X, X) == 1  # T is not 1
    ok.T = 1
    assert step(None, ctypes.byref(ok), None, None, X) == 2 and step(None, ctypes.byref(ok), None, X, None) == 2
    empty = attention(B=0)
    assert fwd(None, ctypes.byref(empty), None, None, None, 0) == 0 and back(empty) == 0


@pytest.mark.parametrize("sfx", SFX)
def test_launches_stay_within_32_bits(lib, sfx):
    """Problems times heads past 2^22, and chunks of the backward pass past 2^31."""
    fwd, bwd = (getattr(lib, f"tmpc_delta_attention_{n}_{sfx}") for n in ("forward", "backward"))
    st, eb = (ctypes.c_int64 * 3)(1, 1, 1), 2 if sfx == "bf16" else 4
    back = lambda a: bwd(None, ctypes.byref(a), X, st, None, X, X, X, X, X, X, None, 0)  # noqa: E731
    most = attention(B=1 << 20, H=4, T=1, **DATA)
    assert fwd(None, ctypes.byref(most), None, None, None, 0) == 2 and back(most) == 3
    more = attention(B=(1 << 20) + 1, H=4, T=1, **DATA)
    assert fwd(None, ctypes.byref(more), X, X, None, 0) == 1 and back(more) == 1
    query = lambda **kw: lib.tmpc_delta_attention_workspace_bytes(eb, ctypes.byref(attention(**kw)), 1)  # noqa: E731
    long = dict(B=64, H=4, T=8388576)  # just below 2^26 chunks
    assert long["B"] * long["H"] * -(-long["T"] // 32) < 1 << 31
    assert back(attention(**long, **DATA)) == 3 and query(**long) > 0
    long = dict(B=1024, H=4, T=1 << 24)
    assert back(attention(**long, **DATA)) == 1 and query(**long) == 0


@pytest.mark.parametrize("eb", [2, 4])
def test_workspaces(lib, eb):
    query = lib.tmpc_delta_attention_workspace_bytes
    sfx = "bf16" if eb == 2 else "f32"
    fwd, bwd = (getattr(lib, f"tmpc_delta_attention_{n}_{sfx}") for n in ("forward", "backward"))
    need = lambda backward=0, **kw: query(eb, ctypes.byref(attention(**kw)), backward)  # noqa: E731
    assert need(B=256, T=512) == 0  # whole histories
    assert need(B=1, T=50000) > 0 and need(B=1, T=50000) % 256 == 0  # runs
    assert need(1) < need(1, T=50) < need(1, T=50, B=64) and need(1, T=50, Hv=4) < need(1, T=50, Hv=2)
    assert need(1, T=0) == 0 and need(1, B=0) == 0
    assert query(3, ctypes.byref(attention()), 1) == 0 and query(eb, ctypes.byref(attention(dk=0)), 1) == 0
    a = attention(B=1, T=50000, **DATA)
    n = query(eb, ctypes.byref(a), 0)
    assert fwd(None, ctypes.byref(a), X, X, X, n - 1) == 3 and fwd(None, ctypes.byref(a), X, X, None, n) == 2
    st = (ctypes.c_int64 * 3)(1, 1, 1)
    n = query(eb, ctypes.byref(a), 1)
    assert bwd(None, ctypes.byref(a), X, st, None, X, X, X, X, X, X, X, n - 1) == 3
    assert bwd(None, ctypes.byref(a), X, st, None, X, X, X, X, X, X, None, n) == 2


def test_host_tensors_are_refused():
    q, g = torch.zeros(1, 3, 2, 8), torch.zeros(1, 3, 2)
    with pytest.raises(ValueError, match="HIP device"):
        learning.delta_attention(q, q, q, g, g)
    with pytest.raises(ValueError, match="HIP device"):
        learning.delta_attention_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], g[:, 0], torch.zeros(1, 2, 8, 8))
    with pytest.raises(TypeError):
        learning.delta_attention(q.double(), q, q, g, g)


def test_model_options_are_checked():
    for bad in (dict(memory="none"), dict(norm="batch"), dict(dropout=1.0), dict(dropout=-0.1)):
        with pytest.raises(ValueError):
            learning.HistoryWeights(5, {"a": 2}, width=16, heads=2, device="cpu", **bad)
    m = learning.HistoryWeights(5, {"a": 2}, width=16, heads=2, device="cpu", dropout=0.1)
    with pytest.raises(ValueError, match="key"):
        m(torch.zeros(1, 3, 5))
    m = learning.HistoryWeights(5, {"a": 2}, width=16, heads=2, device="cpu", memory="delta", norm="layer").bfloat16()
    assert all(p.dtype == torch.bfloat16 for p in m.parameters())
    assert {"norm_out_bias", "blocks.0.w_gates", "blocks.1.norm_ff_bias"} <= set(m.state_dict())
