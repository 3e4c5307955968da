"""The packed kernels with cu_seqlens that are no lengths (tests/test_packed_pieces.py has their
indexes on the host): the C entry points on tensors that lie between others. What lies around the
inputs is NaN and reaches no output, what lies around the outputs and the workspace keeps its
bits."""
from __future__ import annotations

import pytest
import torch

from mamba_metal_scan_amd import _native

pytestmark = pytest.mark.gpu
GUARD = 1 << 16          # elements on either side
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

BAD = [[0, 50, 20, 300], [-5, 50, 700], [290, 10, 295], [0, 1 << 30], [300, 300, 300, 0], [7],
       [0, 130, 130, 131], [40, 35, 30, 25, 20, 300], [0] * 70 + [299, 5]]


class Arena:
    """Tensors between guards."""

    def __init__(self):
        self.made = []

    def _place(self, shape, dtype, fill, guard):
        n = 1
        for s in shape:
            n *= s
        whole = torch.full((2 * GUARD + n + 64,), guard, dtype=dtype, device="cuda")
        t = whole[GUARD:GUARD + n].view(shape)
        t.copy_(fill) if torch.is_tensor(fill) else t.fill_(fill)
        return whole, t

    def input(self, t):
        return self._place(t.shape, t.dtype, t, float("nan"))[1]

    def rows(self, t):
        """t's rows in wider ones, NaN between and around them."""
        wide = torch.full((t.shape[0], t.shape[1] + 8), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, :t.shape[1]] = t
        return self.input(wide)[:, :t.shape[1]]

    def output(self, *shape, dtype=torch.float32, fill=0.5):
        whole, t = self._place(shape, dtype, fill, 77.0)
        self.made.append((whole, t.numel()))
        return t

    def workspace(self, nbytes):
        return self.output(max(64, (nbytes + 3) // 4), fill=0.0)

    def check(self):
        torch.cuda.synchronize()
        for whole, n in self.made:
            assert (whole[:GUARD] == 77.0).all() and (whole[GUARD + n:] == 77.0).all()
            assert not torch.isnan(whole).any()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _ok(rc):
    assert rc == 0, _native.library().mhs_last_error().decode()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cu_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("which", range(len(BAD)))
def test_scan_stays_within(which, cu_dtype, dtype):
    lib, ar = _native.library(), Arena()
    rows, d, n, nseq = 300, 40, 16, len(BAD[which]) - 1
    g = torch.Generator(device="cuda").manual_seed(which)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    cu = torch.tensor(BAD[which], device="cuda").to(cu_dtype)
    x, b, c, dy = (ar.rows(randn(rows, w).to(dtype)) for w in (d, n, n, d))
    dt = ar.rows((0.01 + 0.1 * torch.sigmoid(randn(rows, d))).to(dtype))
    aneg = ar.input(randn(d, n).exp())
    h0, dh = (ar.input(randn(nseq, d, n)) for _ in range(2))
    y = ar.output(rows, d, dtype=dtype)
    h_last = ar.output(nseq, d, n)
    ckpt = ar.output(lib.mhs_packed_ckpt_floats(rows, d, n))
    for wanted in (None, ckpt):
        nbytes = lib.mhs_packed_scan_workspace_bytes(nseq, rows, d, n, 0)
        ws = ar.workspace(nbytes)
        _ok(lib.mhs_packed_scan_fwd(
            TYPES[dtype], _ptr(x), d + 8, _ptr(dt), d + 8, _ptr(aneg), _ptr(b), n + 8, _ptr(c),
            n + 8, _ptr(cu), cu_dtype == torch.int64, _ptr(h0), _ptr(y), _ptr(h_last),
            _ptr(wanted), nseq, rows, d, n, _ptr(ws), nbytes, None))
        ar.check()
    dx, ddt = ar.output(rows, d, dtype=dtype), ar.output(rows, d, dtype=dtype)
    db, dc = ar.output(rows, n, dtype=dtype), ar.output(rows, n, dtype=dtype)
    da, dh0 = ar.output(d, n), ar.output(nseq, d, n)
    nbytes = lib.mhs_packed_scan_workspace_bytes(nseq, rows, d, n, 1)
    ws = ar.workspace(nbytes)
    _ok(lib.mhs_packed_scan_bwd(
        TYPES[dtype], _ptr(x), d + 8, _ptr(dt), d + 8, _ptr(aneg), _ptr(b), n + 8, _ptr(c), n + 8,
        _ptr(cu), cu_dtype == torch.int64, _ptr(h0), _ptr(ckpt), _ptr(dy), d + 8, _ptr(dh),
        _ptr(dx), _ptr(ddt), _ptr(da), _ptr(db), _ptr(dc), _ptr(dh0), nseq, rows, d, n, _ptr(ws), nbytes,
        None))
    ar.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("taps,d", [(4, 40), (8, 33), (1, 64)])
@pytest.mark.parametrize("which", range(len(BAD)))
def test_conv_stays_within(which, taps, d, dtype):
    lib, ar = _native.library(), Arena()
    rows, nseq = 300, len(BAD[which]) - 1
    g = torch.Generator(device="cuda").manual_seed(which)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    cu = torch.tensor(BAD[which], device="cuda")
    x, dout = ar.rows(randn(rows, d)), ar.rows(randn(rows, d))
    w, bias = ar.input(randn(d, taps)), ar.input(randn(d))
    window, dlast = (ar.input(randn(nseq, d, taps - 1)) for _ in range(2))
    out = ar.output(rows, d, dtype=dtype)
    last = ar.output(nseq, d, taps - 1, dtype=dtype)
    _ok(lib.mhs_packed_conv_fwd(TYPES[dtype], _ptr(x), d + 8, _ptr(w), _ptr(bias), 0, _ptr(cu), 1,
                                _ptr(window), _ptr(out), _ptr(last), nseq, rows, d, taps, None))
    ar.check()
    dx, dwin = ar.output(rows, d, dtype=dtype), ar.output(nseq, d, taps - 1, dtype=dtype)
    dw, db = ar.output(d, taps, dtype=dtype), ar.output(d, dtype=dtype)
    nbytes = lib.mhs_packed_conv_bwd_workspace_bytes(nseq, rows, d, taps)
    ws = ar.workspace(nbytes)
    _ok(lib.mhs_packed_conv_bwd(
        TYPES[dtype], _ptr(x), d + 8, _ptr(w), _ptr(bias), 0, _ptr(cu), 1, _ptr(window), _ptr(dout),
        d + 8, _ptr(dlast), _ptr(dx), _ptr(dw), _ptr(db), _ptr(dwin), nseq, rows, d, taps, _ptr(ws),
        nbytes, None))
    ar.check()
