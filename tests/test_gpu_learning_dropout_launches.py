"""Dropout of more pieces than the 2^31 that one launch counts (turbompc_amd.learning): the second launch's rows."""
import numpy as np
import pytest
import torch

import learning_reference_blocks as ref
from turbompc_amd import learning

pytestmark = pytest.mark.gpu
DEV = "cuda"
SEED, STEP, CALL = 0x123456789ABCDEF, 77, 4


def mask(rows, width, p):
    """Which elements of these rows are kept."""
    words = ref.philox((np.arange((width + 7) // 8)[None], rows[:, None], CALL, STEP), (SEED % 2 ** 32, SEED >> 32))
    bits = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=-1)
    return torch.from_numpy(bits.reshape(len(rows), -1)[:, :width].astype(np.int64)) >= round(p * 65536)


@pytest.mark.parametrize("dtype,width", [(torch.float32, 5), (torch.bfloat16, 9)])  # two pieces a row
def test_rows_of_the_second_launch(dtype, width):
    most, p = 1 << 30, 0.25
    M = most + 3000
    row = torch.arange(1, width + 1, dtype=dtype, device=DEV) * 3  # times 4 / 3: exact
    y = learning.dropout(row.expand(M, width), p, torch.tensor([SEED, STEP], device=DEV), CALL)
    assert y.shape == (M, width)
    for r0, r1 in ((0, 50), (most // 2 - 20, most // 2 + 20), (most - 50, most + 50), (M - 2000, M)):
        want = torch.where(mask(np.arange(r0, r1, dtype=np.uint64), width, p), 4.0 * torch.arange(1, width + 1), 0.0)
        assert torch.equal(y[r0:r1].cpu(), want.to(dtype)), r0
    del y
    torch.cuda.empty_cache()
