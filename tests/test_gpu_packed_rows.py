"""The packed scan of nearly 2^31 rows, all one sequence: its pieces are counted without passing 32 bits."""
from __future__ import annotations

import pytest
import torch

from mamba_metal_scan_amd import selective_scan_packed

pytestmark = pytest.mark.gpu


def test_one_sequence_of_nearly_all_rows():
    """One channel of one state that keeps what it has (Aneg 0): the first row's 1 is in every y,
    through two million pieces."""
    rows = 2 ** 31 - 200
    one = torch.ones(rows, 1, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros_like(one)
    x[0] = 1
    aneg = torch.zeros(1, 1, device="cuda")
    cu = torch.tensor([0, rows], device="cuda")
    y, h = selective_scan_packed(x, one, aneg, one, one, cu, return_state=True)
    assert float(h) == 1.0
    assert int((y != 1).sum()) == 0
