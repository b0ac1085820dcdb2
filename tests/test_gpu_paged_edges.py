"""Paged block memory on the GPU: calls at the edges of what its documentation
allows.  Tolerances as in test_gpu_paged.py (``Setup.check``)."""
import numpy as np
import pytest
import torch

from test_gpu_paged import BF16, FP16, Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, d, G", [(BF16, 128, 1), (FP16, 64, 1), (BF16, 64, 2), (FP16, 128, 2)])
def test_many_one_tile_parts_of_few_rows_in_a_row(cuda_device, dtype, d, G):
    # a worker takes some dozen parts of one or two rows and one tile each, one
    # right behind the other: no row takes its neighbour's references and sums
    rng = np.random.default_rng(G)
    lens = rng.integers(1, 129, 1500)
    s = Setup(cuda_device, dtype, lens, [1] * 1500, 0, 2, G, d, 64, seed=d + G)
    out, lse = s.run()
    s.check(out, lse)
    for _ in range(5):
        again, lse2 = s.run()
        assert torch.equal(out, again) and torch.equal(lse, lse2)
