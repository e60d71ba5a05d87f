"""The layer norm and dropout without a GPU: the generator's published answers, what the C entry
points and the Python layer refuse before anything is enqueued."""
import ctypes

import pytest
import torch

import learning_reference_blocks as ref
from turbompc_amd import _lib, learning

SFX = ["f32", "bf16"]
X = ctypes.c_void_p(0x1000)  # never read: every call below returns before a launch


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_generator_against_its_published_answers():
    """The known answers that the generator's authors give for ten rounds."""
    for counter, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((2 ** 32 - 1,) * 4, (2 ** 32 - 1,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(w) for w in ref.philox(counter, key)) == want


@pytest.mark.parametrize("sfx", SFX)
def test_dropout_refusals(lib, sfx):
    f = getattr(lib, f"tmpc_dropout_{sfx}")
    for rows, width in ((-1, 8), (2 ** 31, 8), (4, 0), (4, 2 ** 24 + 1)):
        assert f(None, rows, width, X, 8, 0.5, X, 0, X) == 1
    for p in (-0.1, 1.0, 1.0 - 2.0 ** -18, float("nan"), float("inf")):
        assert f(None, 4, 8, X, 8, p, X, 0, X) == 2, p
    assert f(None, 4, 8, None, 8, 0.5, X, 0, X) == 2
    assert f(None, 4, 8, X, 8, 0.5, None, 0, X) == 2
    assert f(None, 4, 8, X, 8, 0.5, X, 0, None) == 2
    assert f(None, 4, 8, X, -8, 0.5, X, 0, X) == 2
    assert f(None, 0, 8, None, 8, 0.5, None, 0, None) == 0


@pytest.mark.parametrize("sfx", SFX)
def test_layer_norm_refusals(lib, sfx):
    fwd, bwd = (getattr(lib, f"tmpc_layer_norm_{n}_{sfx}") for n in ("forward", "backward"))
    full = dict(rows=4, width=8, call=0, x=X.value, residual=None, weight=X.value, bias=None, ldx=8, ldr=0, eps=1e-5,
                p=0.0, key=None)
    make = lambda **kw: ctypes.byref(_lib.LayerNorm(**{**full, **kw}))  # noqa: E731
    back = lambda a, ws=X, n=1 << 40: bwd(None, a, X, 8, None, 0, X, 8, X, X, None, X, None, ws, n)  # noqa: E731
    for bad in (dict(rows=-1), dict(width=0), dict(width=8193), dict(rows=2 ** 31, p=0.5, key=X.value)):
        assert fwd(None, make(**bad), X, X, X) == 1, bad
        assert back(make(**bad)) == 1, bad
    assert fwd(None, None, X, X, X) == 1
    for bad in (dict(weight=None), dict(p=0.5), dict(p=1.0, key=X.value), dict(p=-0.5, key=X.value),
                dict(p=float("nan"), key=X.value)):
        assert fwd(None, make(**bad), X, X, X) == 2, bad
        assert back(make(**bad)) == 2, bad
    for bad in (dict(x=None), dict(eps=-1.0), dict(eps=float("nan")), dict(ldx=-1), dict(ldr=-1)):
        assert fwd(None, make(**bad), X, X, X) == 2, bad
    assert fwd(None, make(), None, X, X) == 2 and fwd(None, make(), X, None, X) == 2
    eb = 2 if sfx == "bf16" else 4
    need = lib.tmpc_layer_norm_backward_workspace_bytes(eb, 4, 8)
    assert need > 0
    assert back(make(), X, 63) == 3
    assert back(make(), None, need) == 2
    assert fwd(None, make(rows=0, x=None, weight=None), None, None, None) == 0
    assert lib.tmpc_layer_norm_backward_workspace_bytes(3, 4, 8) == 0


def test_host_tensors_and_wrong_types_are_refused():
    x, w = torch.zeros(2, 8), torch.zeros(8)
    key = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: learning.dropout(x, 0.5, key), lambda: learning.layer_norm_residual(x, None, w)):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    for call in (lambda: learning.dropout(x.double(), 0.5, key), lambda: learning.dropout(None, 0.5, key),
                 lambda: learning.layer_norm_residual(x.half(), None, w)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("p", [float("inf"), -float("inf"), float("nan"), 1e300, 1.0, 1.0 - 2.0 ** -18, -1e-9])
def test_probabilities_out_of_range_are_value_errors(p):
    from turbompc_amd.learning.norm_ops import _check_dropout

    with pytest.raises(ValueError, match="at least 0"):
        _check_dropout(torch.zeros(2, 8), p, torch.zeros(2, dtype=torch.int64), 0, "p")
