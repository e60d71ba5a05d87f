"""How the gated delta rule cuts long histories into runs, by its workspace query (no GPU): whole histories need
no workspace forwards, a run's state and map are whole tiles of floats."""
import ctypes

import pytest

from turbompc_amd import _lib


def runs(B, H, T, d):
    """The runs of each of the B H histories of T steps, d wide."""
    a = _lib.DeltaAttention(B=B, T=T, H=H, Hq=H, Hk=H, Hv=H, dk=d, dv=d)
    n = _lib.load().tmpc_delta_attention_workspace_bytes(4, ctypes.byref(a), 0)
    size = B * H * 2 * d * d * 4
    assert n % size == 0
    return n // size or 1


@pytest.mark.parametrize("d", [32, 64, 128])
def test_no_history_is_cut_into_two(d):
    """Four runs or more are wanted, or one; whole stretches of 256 steps can come out as three."""
    seen = set()
    for heads in (1, 2, 5, 16, 32, 48, 63, 64, 65, 85, 100, 127, 128, 129, 200, 512):
        for T in range(1, 12000, 128):
            n = runs(1, heads, T, d)
            seen.add(n)
            assert n != 2 and (n != 3 or -(-T // 256) in (5, 6, 9)) and (n == 1 or heads <= 128), (heads, T, n)
    assert 1 in seen and max(seen) > 8


def test_long_histories_of_few_heads_are_cut():
    assert runs(1, 128, 1024, 64) == 4 and runs(2, 8, 50000, 128) > 8 and runs(1, 1, 1025, 64) == 5
    assert runs(1, 129, 50000, 64) == 1 and runs(1, 65, 50000, 128) == 1 and runs(256, 4, 100000, 64) == 1
