"""Sampling of rows that the first kernel leaves to the others, one for each way that they go: the parts'
sums, the bins, the search for k, and +inf among the words, all in one call."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_sample import _rand, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_left_to_each_kernel(dtype):
    z, u = _rand(10, 20001, dtype, 31)
    z[5:7, ::2] = math.inf       # 10001 words that share the draw
    k = torch.tensor([0, 5000, 5000, 0, 3000, 0, 0, 4000, 20000, 20001])
    p = torch.tensor([1.0, 1.0, 0.9, 0.9, 1.0, 1.0, 0.7, 1.0, 1.0, 0.99])
    low = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.001, 0.0, 0.0, 0.0, 0.0, 0.0])
    z[7, 3::4] = -math.inf
    check(z, u, top_k=k, top_p=p, min_p=low)
    check(z, u, top_k=k, min_p=low)
