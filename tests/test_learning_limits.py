"""Limits of the history model's C entry points, without a GPU: a call past one is refused
before anything is enqueued."""
import ctypes

import pytest

from turbompc_amd import _lib

X = ctypes.c_void_p(0x1000)  # never read: every call below returns before a launch


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("sfx,elem_bytes", [("f32", 4), ("bf16", 2)])
@pytest.mark.parametrize("H", [1, 3, 256])
def test_steps_whose_runs_pass_31_bits(lib, H, sfx, elem_bytes):
    """A kernel counts steps in 32 bits, up to the end of the last run of whole chunks:
    more than 2^30 steps are refused."""
    def args(T):
        return _lib.DecayAttention(B=1, T=T, H=H, Hk=H, dk=1, dv=1, q=X.value, k=X.value, v=X.value, log_decay=X.value,
                                   q_stride=(0, 1, 1), k_stride=(0, 1, 1), v_stride=(0, 1, 1), scale=1.0)

    stride = (ctypes.c_int64 * 3)(0, 1, 1)
    for T in (2 ** 30 + 1, 2 ** 31 - 64, 2 ** 31 - 1):
        a = args(T)
        assert getattr(lib, f"tmpc_decay_attention_forward_{sfx}")(None, ctypes.byref(a), X, X, X, 1 << 40) == 1, T
        assert getattr(lib, f"tmpc_decay_attention_backward_{sfx}")(None, ctypes.byref(a), X, stride, None, X, X, X, None,
                                                                   X, 1 << 40) == 1, T
        for backward in (0, 1):
            assert lib.tmpc_decay_attention_workspace_bytes(elem_bytes, ctypes.byref(a), backward) == 0, T
    # the longest history that is taken asks for the runs' states as before
    need = lib.tmpc_decay_attention_workspace_bytes(elem_bytes, ctypes.byref(args(2 ** 30)), 0)
    assert (need > 0) == (H < 256)
