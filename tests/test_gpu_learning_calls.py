"""What a caller of the history model's operators may count on beside the values: limits,
views, torch's autograd rules."""
import pytest
import torch

from turbompc_amd import learning

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]


def test_histories_past_the_step_limit_are_refused():
    q = torch.zeros((1, 1, 1, 1), device=DEV)
    g = torch.zeros(1, device=DEV)
    for T in (2 ** 30 + 1, 2 ** 31):
        x = q.expand(1, T, 1, 1)  # no memory behind it
        with pytest.raises(ValueError):
            learning.decay_attention(x, x, x, g)
