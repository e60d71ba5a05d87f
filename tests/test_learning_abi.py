"""The history model's C entry points and Python checks without a GPU: what they refuse
before anything is enqueued, and the workspace queries."""
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
    a = dict(B=2, T=5, H=4, Hk=2, dk=16, dv=16)
    a.update(kw)
    return _lib.DecayAttention(**a)


@pytest.mark.parametrize("sfx", SFX)
def test_attention_refusals(lib, sfx):
    fwd, bwd, step = (getattr(lib, f"tmpc_decay_attention_{n}_{sfx}") for n in ("forward", "backward", "step"))
    for bad in (dict(H=3), dict(dk=0), dict(dk=129), dict(dv=129), dict(B=-1), dict(T=-1), dict(Hk=0), dict(H=0),
                dict(B=2 ** 30)):
        a = attention(**bad)
        assert fwd(None, ctypes.byref(a), X, X, None, 0) == 1, bad
        assert bwd(None, ctypes.byref(a), X, None, X, X, X, X, X, None, 0) == 1, bad
        a.T = 1 if "T" not in bad else a.T
        assert step(None, ctypes.byref(a), None, X, X) == 1, bad
    assert fwd(None, None, X, X, None, 0) == 1
    ok = attention()
    assert fwd(None, ctypes.byref(ok), X, X, None, 0) == 2  # no data
    assert bwd(None, ctypes.byref(ok), X, None, X, X, X, X, X, None, 0) == 2
    assert step(None, ctypes.byref(ok), None, X, X) == 1  # T is not 1
    assert step(None, ctypes.byref(attention(T=1)), None, X, X) == 2
    empty = attention(B=0)
    assert fwd(None, ctypes.byref(empty), None, None, None, 0) == 0
    full = attention(q=X.value, k=X.value, v=X.value, log_decay=X.value)
    need = lib.tmpc_decay_attention_workspace_bytes(2 if sfx == "bf16" else 4, ctypes.byref(full), 1)
    st = (ctypes.c_int64 * 3)(1, 1, 1)
    assert need > 0
    assert bwd(None, ctypes.byref(full), X, st, None, X, X, X, None, X, need - 1) == 3
    assert bwd(None, ctypes.byref(full), X, st, None, X, X, X, None, None, need) == 2


@pytest.mark.parametrize("sfx", SFX)
def test_feed_forward_refusals(lib, sfx):
    fwd, bwd = (getattr(lib, f"tmpc_gated_ff_{n}_{sfx}") for n in ("forward", "backward"))
    full = dict(M=4, D=8, F=8, Dout=8, activation=0, x=X.value, ldx=8, w_gate=X.value, w_up=X.value, w_down=X.value)
    make = lambda **kw: ctypes.byref(_lib.GatedFF(**{**full, **kw}))  # noqa: E731
    for bad in (dict(M=-1), dict(D=0), dict(F=0), dict(Dout=0), dict(M=2 ** 31)):
        assert fwd(None, make(**bad), X, None, None, X, 1 << 40) == 1, bad
        assert bwd(None, make(**bad), X, X, X, 8, X, X, X, X, X, 1 << 40) == 1, bad
    for bad in (dict(activation=2), dict(x=None), dict(w_up=None), dict(ldx=-1)):
        assert fwd(None, make(**bad), X, None, None, X, 1 << 40) == 2, bad
        assert bwd(None, make(**bad), X, X, X, 8, X, X, X, X, X, 1 << 40) == 2, bad
    assert fwd(None, make(), X, X, None, X, 1 << 40) == 2  # one projection alone
    eb = 2 if sfx == "bf16" else 4
    need = lib.tmpc_gated_ff_workspace_bytes(eb, make(), 0)
    assert 0 < need <= lib.tmpc_gated_ff_workspace_bytes(eb, make(), 1)
    assert fwd(None, make(), X, None, None, X, need - 1) == 3
    assert bwd(None, make(), X, X, X, 8, X, X, X, X, X, need - 1) == 3
    assert fwd(None, make(M=0), None, None, None, None, 0) == 0
    for backward in (0, 1):  # an empty batch has a workspace query too
        assert lib.tmpc_gated_ff_workspace_bytes(eb, make(M=0), backward) == 0


@pytest.mark.parametrize("sfx", SFX)
def test_norm_refusals(lib, sfx):
    fwd, bwd = (getattr(lib, f"tmpc_rms_norm_{n}_{sfx}") for n in ("forward", "backward"))
    for rows, width in ((-1, 8), (4, 0), (4, 8193)):
        assert fwd(None, rows, width, X, 8, None, 0, X, 1e-6, X, X, X) == 1
        assert bwd(None, rows, width, X, 8, None, 0, X, 8, X, X, X, X, X, 1 << 40) == 1
    assert fwd(None, 4, 8, None, 8, None, 0, X, 1e-6, X, X, X) == 2
    assert fwd(None, 4, 8, X, 8, None, 0, X, -1.0, X, X, X) == 2
    assert fwd(None, 4, 8, X, 8, None, 0, X, float("nan"), X, X, X) == 2
    assert fwd(None, 0, 8, None, 8, None, 0, None, 1e-6, None, None, None) == 0
    eb = 2 if sfx == "bf16" else 4
    need = lib.tmpc_rms_norm_backward_workspace_bytes(eb, 1000, 64)
    assert need > 0
    assert bwd(None, 1000, 64, X, 64, None, 0, X, 64, X, X, X, X, X, 255) == 3


def test_host_tensors_are_refused():
    q = torch.zeros(1, 3, 2, 8)
    with pytest.raises(ValueError):
        learning.decay_attention(q, q, q, torch.zeros(2))
    with pytest.raises(ValueError):
        learning.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(2), torch.zeros(1, 2, 8, 8))
    w = torch.zeros(4, 8)
    with pytest.raises(ValueError):
        learning.gated_feed_forward(torch.zeros(2, 8), w, w, w.t())
    with pytest.raises(ValueError):
        learning.rms_norm_residual(torch.zeros(2, 8), None, torch.zeros(8))
    with pytest.raises(TypeError):
        learning.rms_norm_residual(torch.zeros(2, 8, dtype=torch.float64), None, torch.zeros(8))
