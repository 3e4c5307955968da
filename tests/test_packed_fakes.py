"""The registered packed operators under tracing: shapes, types and devices of their outputs without
running them, for every layout of the weights and every output that may be left out, as the kernels
give them."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mamba_metal_scan_amd  # noqa: F401  (registers the operators)
from mamba_metal_scan_amd import conv1d_silu_packed

OPS = torch.ops.mamba_hip
ROWS, D, SEQS = 16, 4, 2


def _conv_args(taps, three, dtype, device):
    g = torch.Generator().manual_seed(taps)
    x = torch.randn(ROWS, D, generator=g).to(dtype).to(device)
    w = torch.randn(D, taps, generator=g).to(dtype).to(device)
    bias = torch.randn(D, generator=g).to(dtype).to(device)
    cu = torch.tensor([0, 5, ROWS], device=device)
    window = torch.randn(SEQS, D, taps - 1, generator=g).to(dtype).to(device)
    return x, w.view(D, 1, taps) if three else w, bias, cu, window


def _conv(taps, three, dtype, with_window, device):
    """(outputs of the forward, of the backward)"""
    x, w, bias, cu, window = _conv_args(taps, three, dtype, device)
    window = window if with_window else None
    fwd = OPS.packed_conv_fwd(x, w, bias, cu, window, True)
    bwd = OPS.packed_conv_bwd(x, w, bias, cu, window, torch.ones_like(x), torch.ones_like(fwd[1]))
    return fwd, bwd, OPS.packed_conv_fwd(x, w, bias, cu, window, False)


def _like(t):
    return tuple(t.shape), t.dtype


CASES = [(taps, three, with_window) for taps in (1, 4, 8) for three in (False, True)
         for with_window in (False, True)]


@pytest.mark.parametrize("taps,three,with_window", CASES)
def test_conv_shapes_of_either_weight(taps, three, with_window):
    f = torch.float32
    with FakeTensorMode():
        fwd, bwd, without = _conv(taps, three, f, with_window, "cuda")
    wshape = (D, 1, taps) if three else (D, taps)
    assert [_like(t) for t in fwd] == [((ROWS, D), f), ((SEQS, D, taps - 1), f)]
    assert [_like(t) for t in without] == [((ROWS, D), f), ((0,), f)]
    assert [_like(t) for t in bwd] == [((ROWS, D), f), (wshape, f), ((D,), f),
                                       ((SEQS, D, taps - 1) if with_window else (0,), f)]


@pytest.mark.gpu
@pytest.mark.parametrize("taps,three,with_window", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_conv_fakes_are_as_the_kernels(taps, three, with_window, dtype):
    real = _conv(taps, three, dtype, with_window, "cuda")
    with FakeTensorMode():
        fake = _conv(taps, three, dtype, with_window, "cuda")
    for a, b in zip(real, fake):
        assert [(_like(t), t.stride(), t.device) for t in a] == \
            [(_like(t), t.stride(), t.device) for t in b]


@pytest.mark.gpu
@pytest.mark.parametrize("three", [False, True])
def test_conv_traced_with_its_windows(three):
    x, w, bias, cu, window = _conv_args(4, three, torch.float32, "cuda")

    def f(x, w, bias, window):
        return conv1d_silu_packed(x, w, bias, cu, window=window, return_window=True)

    leaves = [t.requires_grad_(True) for t in (x, w, bias, window)]
    want = f(*leaves)
    ups = [torch.randn_like(t) for t in want]
    grads = torch.autograd.grad(want, leaves, ups)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(torch.autograd.grad(got, leaves, ups), grads):
        assert torch.equal(a, b)
