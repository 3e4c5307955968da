"""Sampling of rows whose largest logit is -0, before or behind the words that lie in whole vectors:
it counts as 0, and has its place in the order by that."""
from __future__ import annotations

import pytest
import torch

from test_gpu_sample import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,least", [(torch.float32, 2.0 ** -149), (torch.bfloat16, 2.0 ** -133)])
@pytest.mark.parametrize("zero", [-0.0, 0.0])
def test_a_largest_logit_of_minus_zero(zero, dtype, least):
    """All other words one step below 0, each of weight 1: of 2003 words that start or end outside
    a 16-byte vector the 300 first, and a number in the 299th word's share."""
    z = torch.full((2, 2003), -least, dtype=dtype)
    assert float(z[0, 0]) == -least
    z[0, 2002] = zero      # row 0 is aligned and ends in single words, row 1 begins with some
    z[1, 0] = zero
    u = torch.full((2,), 0.995)
    for s in (dict(top_k=300), dict(top_k=300, top_p=0.9), dict(top_k=500, min_p=0.5), dict(),
              dict(top_p=0.5), dict(temperature=0.0), dict(top_k=1)):
        check(z, u, **s)
