"""The kernels' variants by size (turbompc_amd.learning) at shapes that take each of them, against
the definitions in 64 bits."""
import pytest
import torch

import learning_reference as ref
from test_gpu_learning_blocks import DTYPES, ff_inputs, ff_run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(4400, 72, 2200, 72), (4400, 2056, 72, 2056), (4400, 200, 2201, 40),
                                   (2600, 72, 2200, 72), (1100, 512, 520, 520)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", DTYPES)
def test_feed_forward_forms_by_size(shape, dtype):
    """More tiles of 256 than half the CUs (each product in turn, where rows are whole pieces), tiles of
    128 and of 64."""
    x = ff_inputs(*shape, dtype, seed=sum(shape))
    got = ff_run(x, "gelu")
    for k, (v, tol) in ref.feed_forward(x["x"], x["wg"], x["wu"], x["wd"], "gelu", x["dy"]).items():
        ref.assert_within(k, got[k], v, tol)
