"""The packed operators' refusals without a GPU: tensors elsewhere and bad arguments raise before any
call, and the C entry points return MHS_EINVAL (fake addresses: nothing is launched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import mamba_metal_scan_amd as m
from mamba_metal_scan_amd import _native
from mamba_metal_scan_amd._native import HipScanError

OPS = torch.ops.mamba_hip


def _scan(rows=6, d=4, n=3):
    return (torch.randn(rows, d), torch.rand(rows, d), torch.rand(d, n), torch.randn(rows, n),
            torch.randn(rows, n))


def test_cpu_tensors_are_refused():
    cu = torch.tensor([0, 6])
    x, w, b = torch.randn(6, 4), torch.randn(4, 3), torch.randn(4)
    for call in (lambda: m.selective_scan_packed(*_scan(), cu),
                 lambda: m.conv1d_silu_packed(x, w, b, cu),
                 lambda: m.conv1d_silu_step(x, w, b, torch.zeros(6, 4, 2)),
                 lambda: m.selective_state_step_slots(torch.zeros(6, 4, 3), *_scan()),
                 lambda: m.sample_tokens(x, torch.rand(6))):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()
    with pytest.raises(HipScanError, match="one ROCm device"):
        OPS.packed_scan_fwd(*_scan(), cu, None, True, False)
    with pytest.raises(HipScanError, match="one ROCm device"):
        OPS.packed_conv_fwd(x, w, b, cu, None, False)
    with pytest.raises(HipScanError, match="one ROCm device"):
        OPS.conv_step(x, w, b, torch.zeros(6, 4, 2), None)
    with pytest.raises(HipScanError, match="one ROCm device"):
        OPS.state_step(torch.zeros(6, 4, 3), *_scan(), None)
    with pytest.raises(HipScanError, match="one ROCm device"):
        OPS.sample(x, torch.rand(6), None, None, None, None, [1.0, 1.0, 0.0], 0)


A = ctypes.c_void_p(0x7F0000001000)     # 256-byte aligned
MIS = ctypes.c_void_p(0x7F0000001004)
F32 = 0

# Fake addresses: only where no GPU could be reached by a regression in the checks.
cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device addresses")


def _err():
    return _native.library().mhs_last_error().decode()


def _packed_scan(dtype=F32, x=A, ld=64, aneg=A, cu=A, h0=None, nseq=3, total=100, d=64, n=16,
                 ld_b=16, ws=A, nbytes=1 << 40):
    return _native.library().mhs_packed_scan_fwd(
        dtype, x, ld, A, 64, aneg, A, ld_b, A, 16, cu, 0, h0, A, None, None, nseq, total, d, n, ws,
        nbytes, None)


@cpu_only
def test_packed_scan_arguments():
    for kw, text in ((dict(dtype=7), "dtype"), (dict(x=None), "null"), (dict(aneg=None), "null"),
                     (dict(cu=None), "null"), (dict(ld=63), "rows of x"),
                     (dict(ld=1 << 18), "rows of x"), (dict(ld_b=15), "rows of B"),
                     (dict(h0=MIS), "aligned"), (dict(n=0), "d_state"), (dict(n=65), "d_state"),
                     (dict(d=0), "channels"), (dict(d=(1 << 17) + 1), "channels"),
                     (dict(total=-1), "rows"), (dict(total=1 << 31), "rows"),
                     (dict(nseq=-1), "sequences"), (dict(nseq=(1 << 22) + 1), "sequences"),
                     (dict(nseq=1 << 22, n=16), "too many"), (dict(ws=None), "workspace"),
                     (dict(nbytes=16), "workspace"), (dict(ws=MIS), "256")):
        assert _packed_scan(**kw) == 1, kw
        assert text in _err(), (kw, _err())
    lib = _native.library()
    assert lib.mhs_packed_scan_workspace_bytes(3, 100, 64, 65, 0) == 0
    # up to 64 rows no sequence is longer than a piece: no carries
    assert lib.mhs_packed_scan_workspace_bytes(3, 64, 64, 16, 0) == 0
    assert lib.mhs_packed_scan_workspace_bytes(3, 65, 64, 16, 0) > 0
    assert lib.mhs_packed_ckpt_floats(100, 64, 16) == 12 * 64 * 16


@cpu_only
def test_packed_scan_backward_arguments():
    lib = _native.library()

    def call(ckpt=A, dy=A, da=A, ws=A, nbytes=1 << 40, ld_dy=64):
        return lib.mhs_packed_scan_bwd(F32, A, 64, A, 64, A, A, 16, A, 16, A, 0, None, ckpt, dy,
                                       ld_dy, None, A, A, da, A, A, None, 3, 100, 64, 16, ws,
                                       nbytes, None)

    for kw, text in ((dict(ckpt=None), "null"), (dict(dy=None), "null"), (dict(da=None), "null"),
                     (dict(ckpt=MIS), "aligned"), (dict(ld_dy=1), "rows of dy"),
                     (dict(ws=None), "workspace")):
        assert call(**kw) == 1 and text in _err(), (kw, _err())


@cpu_only
def test_conv_and_step_arguments():
    lib = _native.library()

    def conv(dtype=F32, x=A, ld=64, w=A, cu=A, d=64, k=4, total=100, nseq=2):
        return lib.mhs_packed_conv_fwd(dtype, x, ld, w, A, 0, cu, 0, None, A, None, nseq, total, d,
                                       k, None)

    for kw, text in ((dict(dtype=3), "dtype"), (dict(x=None), "null"), (dict(w=None), "null"),
                     (dict(cu=None), "null"), (dict(ld=8), "rows of x"), (dict(k=0), "taps"),
                     (dict(k=9), "taps"), (dict(d=0), "channels"), (dict(total=-5), "rows")):
        assert conv(**kw) == 1 and text in _err(), (kw, _err())

    def step(x=A, rows=4, pool=8, d=64, k=4, slots=A, window=A, ld=64):
        return lib.mhs_conv_step(F32, x, ld, A, A, 0, window, slots, 0, A, rows, pool, d, k, None)

    for kw, text in ((dict(x=None), "null"), (dict(window=None), "null"), (dict(k=9), "taps"),
                     (dict(slots=None, rows=9), "without slots"), (dict(rows=-1), "rows"),
                     (dict(d=0), "channels"), (dict(ld=1), "rows of x")):
        assert step(**kw) == 1 and text in _err(), (kw, _err())
    assert step(rows=0) == 0

    def state(h=A, x=A, aneg=A, rows=4, pool=8, d=64, n=16, ld=64):
        return lib.mhs_state_step(F32, h, x, ld, A, 64, aneg, A, 64, A, 64, A, 0, A, rows, pool, d,
                                  n, None)

    for kw, text in ((dict(h=None), "null"), (dict(x=None), "null"), (dict(h=MIS), "aligned"),
                     (dict(aneg=MIS), "aligned"), (dict(n=65), "d_state"),
                     (dict(pool=1 << 31), "entries"), (dict(ld=3), "rows of x")):
        assert state(**kw) == 1 and text in _err(), (kw, _err())
    assert state(rows=0) == 0


@cpu_only
def test_sample_arguments():
    lib = _native.library()

    def call(dtype=F32, z=A, ld=1000, u=A, tokens=A, rows=4, vocab=1000, ws=A, nbytes=1 << 40,
             top_k=None, k=0):
        return lib.mhs_sample(dtype, z, ld, u, None, 1.0, top_k, 0, k, None, 1.0, None, 0.0, tokens,
                              None, rows, vocab, ws, nbytes, None)

    for kw, text in ((dict(dtype=5), "dtype"), (dict(z=None), "null"), (dict(u=None), "null"),
                     (dict(tokens=None), "null"), (dict(ld=999), "apart"),
                     (dict(rows=1 << 16), "rows"), (dict(vocab=0), "vocab"),
                     (dict(vocab=(1 << 24) + 1, ld=1 << 25), "vocab"),
                     (dict(vocab=5000, ld=5000, ws=None), "workspace"),
                     (dict(vocab=5000, ld=5000, nbytes=8), "workspace"),
                     (dict(vocab=5000, ld=5000, ws=MIS), "256")):
        assert call(**kw) == 1 and text in _err(), (kw, _err())
    assert call(rows=0) == 0
    size = lib.mhs_sample_workspace_bytes
    assert size(4, 4096, 1, 0) == 0                      # all words fit one list
    assert 0 < size(4, 100000, 0, 50) < size(4, 100000, 1, 0) == size(4, 100000, 0, 0)


def test_sample_settings_of_wrong_shapes():
    z, u = torch.randn(4, 10), torch.rand(4)
    if torch.cuda.is_available():
        z, u = z.cuda(), u.cuda()
        for kw in (dict(temperature=torch.ones(3, device="cuda")),
                   dict(top_k=torch.ones(4, device="cuda")),
                   dict(top_p=torch.ones(4, device="cuda", dtype=torch.int64)),
                   dict(min_p=torch.ones(4, 1, device="cuda"))):
            with pytest.raises(ValueError, match="must be a number or a tensor"):
                m.sample_tokens(z, u, **kw)
        with pytest.raises(ValueError, match="logits must be"):
            m.sample_tokens(z, u[:3])
