"""GPU: layer norm of rows whose mean lies halfway between two fp32 numbers."""

import numpy as np
import pytest
import torch

from saeflow_amd import kernels
from test_gpu_norm import check_held

pytestmark = pytest.mark.gpu

# (widths whose rounded inverse moves the mean of the row off the middle; m is below 2^24, where fp32 numbers are 1 apart)
TIES = [(784, 16764789), (1568, 16724867), (3136, 16761403), (4800, 16714346), (6272, 16761403), (12544, 16761403)]


@pytest.mark.parametrize("D,m", TIES)
def test_a_mean_halfway_between_two_numbers_rounds_to_even(D, m):
    """Half of the row is m, half m + 1: the sum is exact, and the mean m + 1/2 rounds to the even one of the two, which decides
    every element of x - mean, and with it every code."""
    row = torch.full((D,), float(m))
    row[1::2] = float(m + 1)
    x = torch.stack([row, torch.randn(D), -row])
    even = float(np.float32(m + 0.5))
    assert even % 2 == 0 and float(np.float32((D * (m + 0.5)) * (1.0 / D))) != even
    want = torch.tensor([even, -even])
    for out_dtype in (torch.float32, torch.bfloat16):
        y, held, mean, rstd = kernels.layer_norm_held(x.cuda(), out_dtype=out_dtype)
        assert torch.equal(mean[[0, 2]].cpu(), want)
        check_held(x, held)
