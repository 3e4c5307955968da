"""The packed scan with decay rates that are infinite: a state that keeps nothing of the row before.
Steps that the kernels walk behind a sequence's last row must leave it as it is, whatever the
length. (The gradient of dt is Aneg times 0 there, NaN by the formula: not compared.)"""
from __future__ import annotations

import math

import pytest
import torch

import packed_reference as ref
from mamba_metal_scan_amd import selective_scan_packed, selective_state_step_slots
from test_gpu_packed import _cu, _d, scan_inputs

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _rates(aneg):
    """Some states of some channels; the channels that have none."""
    d, n = aneg.shape
    with torch.no_grad():
        aneg[0] = math.inf
        aneg[d // 2, n - 1] = math.inf
        aneg[d - 1, 0] = math.inf
    return [c for c in range(d) if c not in (0, d // 2, d - 1)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d,n", [(40, 16), (33, 16), (12, 1), (20, 3), (24, 8), (18, 24), (16, 64)])
@pytest.mark.parametrize("lens", [[5, 0, 1, 16, 17, 8, 24, 31, 9], [130, 15], [333]])
def test_infinite_rates(lens, d, n, dtype):
    ts = scan_inputs(lens, 2, d, n, dtype, True, True)
    finite = _rates(ts[2])
    y, h = selective_scan_packed(*ts[:5], _cu(lens), h0=ts[5], return_state=True)
    rs = [_d(t) for t in ts]
    yr, hr = ref.scan(*rs[:5], lens, rs[5])
    bar = ref.fp32_bar(max(lens), n)
    ref.check("y", y, yr.detach(), bar)
    ref.check("h_last", h, hr.detach(), bar)
    g = torch.Generator().manual_seed(1)
    dy, dh = torch.randn(y.shape, generator=g).to(dtype), torch.randn(h.shape, generator=g)
    got = torch.autograd.grad([y, h], ts, [dy.cuda(), dh.cuda()])
    want = torch.autograd.grad([yr, hr], rs, [dy.double(), dh.double()])
    for name, a, b, terms in zip(("dx", "ddt", "dAneg", "dB", "dC", "dh0"), got, want,
                                 (n, n, sum(lens), d, d, 1)):
        if name == "ddt":
            a, b = a[:, finite], b[:, finite]
        ref.check(name, a, b, ref.fp32_bar(2 * max(lens), terms))
    # without autograd: another kernel
    with torch.no_grad():
        y2, h2 = selective_scan_packed(*ts[:5], _cu(lens), h0=ts[5], return_state=True)
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_a_token_after_it():
    """What the scan leaves, and the state of one more token, as the scan of all of them."""
    lens = [6, 20]
    x, dt, aneg, b, c, _ = scan_inputs(lens, 0, 16, 16, F32, False, False)
    _rates(aneg)
    y, h = selective_scan_packed(x, dt, aneg, b, c, _cu(lens), return_state=True)
    cut = [0, 1, 2, 3, 4] + list(range(6, 25))
    _, pool = selective_scan_packed(x[cut], dt[cut], aneg, b[cut], c[cut], _cu([5, 19]),
                                    return_state=True)
    at = [5, 25]
    out = selective_state_step_slots(pool, x[at], dt[at], aneg, b[at], c[at])
    ref.check("y", out, y[at].double().cpu(), ref.fp32_bar(20, 16))
    ref.check("h", pool, h.double().cpu(), ref.fp32_bar(20, 16))
