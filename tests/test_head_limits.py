"""Sizes and values at the limits of the head's losses, on the CPU (fake device
addresses that fail before any use; only on hosts without a GPU)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mamba_metal_scan_amd import _native

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device addresses")
A = ctypes.c_void_p(0x7F0000001000)
B = ctypes.c_void_p(0x7F0000101000)
EINVAL = 1
HUGE = 1 << 60   # bytes of workspace: never what a call is refused for


def _err():
    return _native.library().mhs_last_error().decode()


def _refused(rc, match):
    assert rc == EINVAL and match in _err(), (rc, _err())


def xent(dtype, rows, vocab, dim):
    """The forward's and the backward's return codes, and the first's message."""
    lib = _native.library()
    fwd = lib.mhs_linear_xent_fwd(dtype, A, dim, A, dim, A, A, A, A, None, A, A, A, rows, vocab,
                                  dim, -100, 1, A, HUGE, None)
    message = _err()
    bwd = lib.mhs_linear_xent_bwd(dtype, A, dim, A, dim, A, A, A, A, None, A, A, A, A, rows,
                                  vocab, dim, 1, A, HUGE, None)
    return fwd, bwd, message


@no_gpu
@pytest.mark.parametrize("dtype,rows,vocab", [
    (0, 1 << 20, 1 << 18),          # 2^24 tiles of 128 x 128, 256 threads each
    (0, 64, 1 << 30), (0, 4, 1 << 30), (1, 4, 1 << 30),   # of 64 words
    (0, 1 << 26, 8), (1, 1 << 26, 8), (2, 1 << 26, 8),    # a wave per row
    (1, 1 << 25, 1 << 19)])         # tiles counted in an int
def test_products_of_more_threads_than_a_launch_counts(dtype, rows, vocab):
    fwd, bwd, message = xent(dtype, rows, vocab, 64)
    assert fwd == EINVAL and "too large" in message and bwd == EINVAL
    lib = _native.library()
    assert lib.mhs_linear_xent_fwd_workspace_bytes(dtype, rows, vocab, 64) == 0
    assert lib.mhs_linear_xent_bwd_workspace_bytes(dtype, rows, vocab, 64) == 0


@pytest.mark.parametrize("dtype,rows,vocab", [(0, 1 << 20, (1 << 18) - 128),
                                              (0, 64, (1 << 30) - 64), (1, 4, (1 << 30) - 64),
                                              (0, (1 << 22) - 4, 8), (1, (1 << 26) - 4, 8),
                                              (1, 1 << 20, 1 << 18)])
def test_the_largest_sizes_are_taken(dtype, rows, vocab):
    lib = _native.library()
    assert lib.mhs_linear_xent_fwd_workspace_bytes(dtype, rows, vocab, 64) > 0
    assert lib.mhs_linear_xent_bwd_workspace_bytes(dtype, rows, vocab, 64) > 0


@no_gpu
def test_distillation_of_more_rows_than_blocks():
    lib = _native.library()
    n = 1 << 24
    _refused(lib.mhs_distill_fwd(0, A, 8, A, A, A, A, A, A, A, A, n, 8, 2, 1.0, 1, A, HUGE, None),
             "2^24")
    _refused(lib.mhs_distill_bwd(0, A, 8, A, A, A, A, A, A, B, n, 8, 2, 1.0, 1, None), "2^24")
    _refused(lib.mhs_linear_distill_fwd(1, A, 8, A, 8, A, A, A, A, A, A, None, A, A, A, n, 8, 8,
                                        2, 1.0, 1, A, HUGE, None), "2^24")
    _refused(lib.mhs_linear_distill_bwd(1, A, 8, A, 8, A, A, A, A, A, None, A, A, A, A, n, 8, 8,
                                        2, 1.0, 1, A, HUGE, None), "2^24")
    assert lib.mhs_distill_workspace_bytes(n) == 0
    assert lib.mhs_distill_workspace_bytes(n - 1) > 0
    assert lib.mhs_distill_workspace_bytes(-1) == 0
