"""The largest launches of the packed operators, on the host: a launch counts its threads in 32 bits,
2^24 blocks of 256, and what would be more is refused by the plan of the direction that runs
(sizes alone, fake addresses: nothing is launched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mamba_metal_scan_amd import _native

A = ctypes.c_void_p(0x7F0000001000)     # 256-byte aligned

# Fake addresses: only where no GPU could be reached by a regression in the checks.
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device addresses")


def _err():
    return _native.library().mhs_last_error().decode()


def _bytes(nseq, total, d, n, back):
    return _native.library().mhs_packed_scan_workspace_bytes(nseq, total, d, n, back)


def _call(back, nseq, total, d, n, ckpt=None):
    """Refused for its sizes, or, these being right, for a null x."""
    lib = _native.library()
    if back:
        rc = lib.mhs_packed_scan_bwd(0, None, d, A, d, A, A, n, A, n, A, 0, None, A, A, d, None, A,
                                     A, A, A, A, None, nseq, total, d, n, A, 16, None)
    else:
        rc = lib.mhs_packed_scan_fwd(0, None, d, A, d, A, A, n, A, n, A, 0, None, A, None, ckpt,
                                     nseq, total, d, n, A, 16, None)
    assert rc == 1
    return _err()


# 512 channels are four blocks of 128. 64 rows are one piece of the forward, 64 // 64 + nseq + 1
# numbers of them, and pieces of 16 rows of the backward, 64 // 16 + nseq + 1.
@pytest.mark.parametrize("seqs,forward,backward", [
    (2 ** 22 - 6, True, True), (2 ** 22 - 5, True, False), (2 ** 22 - 3, True, False),
    (2 ** 22 - 2, False, False)])
def test_short_batches_of_many_sequences(seqs, forward, backward):
    d, n = 512, 1
    assert (4 * (64 // 64 + seqs + 1) < 2 ** 24) == forward
    assert (4 * (64 // 16 + seqs + 1) < 2 ** 24) == backward
    assert (_bytes(seqs, 64, d, n, 1) > 0) == backward
    assert ("too many" in _call(True, seqs, 64, d, n)) == (not backward)
    # with checkpoints the forward asks for its backward too
    assert ("too many" in _call(False, seqs, 64, d, n, ckpt=A)) == (not backward)
    if not forward:
        assert "too many" in _call(False, seqs, 64, d, n)


def test_sums_of_many_rows():
    """dB and dC are summed 256 numbers a block: rows x 2 x N of them."""
    limit = (2 ** 24 - 1) * 256
    for n in (1, 3, 64):
        rows = min(limit // (2 * n), 2 ** 31 - 1)
        assert _bytes(1, rows, 1, n, 1) > 0
        if rows + 1 < 2 ** 31:
            assert "too many" in _call(True, 1, rows + 1, 1, n)
