"""The conv and the scan over packed sequences on the GPU against 64 bits: lengths of zero, one
and many rows, pieces that end inside a sequence, rows behind the last one, odd widths, strides,
types, windows and states in and out, gradients."""
from __future__ import annotations

import pytest
import torch

import packed_reference as ref
from mamba_metal_scan_amd import conv1d_silu_packed, selective_scan_packed

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

LENS = {
    "one": [1],
    "none": [],
    "empty": [0, 0],
    "mixed": [5, 0, 1, 64, 17, 130, 16, 3],
    "long": [333],
    "two_long": [200, 0, 129, 64, 65],
}


def _cu(lens, dtype=torch.int32):
    return torch.tensor([0] + lens, device="cuda").cumsum(0).to(dtype)


def _leaf(t, grad):
    return t.cuda().requires_grad_(grad)


def _d(t):
    return None if t is None else t.detach().double().cpu().requires_grad_(t.requires_grad)


def scan_inputs(lens, pad, d, n, dtype, carried, grad, seed=0):
    g = torch.Generator().manual_seed(seed)
    rows = sum(lens) + pad
    x = torch.randn(rows, d, generator=g).to(dtype)
    dt = (0.001 + 0.1 * torch.rand(rows, d, generator=g)).to(dtype)
    aneg = torch.rand(d, n, generator=g) * n + 0.05
    b_in, c_in = (torch.randn(rows, n, generator=g).to(dtype) for _ in range(2))
    h0 = torch.randn(len(lens), d, n, generator=g) if carried else None
    ts = [_leaf(t, grad) for t in (x, dt, aneg, b_in, c_in)]
    return ts + [_leaf(h0, grad) if carried else None]


def check_scan(lens, pad, d, n, dtype, carried, grad=True, cu_dtype=torch.int32, seed=0):
    ts = scan_inputs(lens, pad, d, n, dtype, carried, grad, seed)
    y, h = selective_scan_packed(*ts[:5], _cu(lens, cu_dtype), h0=ts[5], return_state=True)
    rs = [_d(t) for t in ts]
    yr, hr = ref.scan(*rs[:5], lens, rs[5])
    longest = max(lens, default=0)
    bar = ref.fp32_bar(longest, n)
    ref.check("y", y, yr.detach(), bar)
    ref.check("h_last", h, hr.detach(), bar)
    assert not y[sum(lens):].any()
    if not grad or not sum(lens):
        return
    g = torch.Generator().manual_seed(seed + 1)
    dy = torch.randn(y.shape, generator=g).to(dtype)
    dh = torch.randn(h.shape, generator=g)
    leaves = [t for t in ts if t is not None]
    got = torch.autograd.grad([y, h], leaves, [dy.cuda(), dh.cuda()])
    want = torch.autograd.grad([yr, hr], [t for t in rs if t is not None],
                               [dy.double(), dh.double()])
    for name, a, b, terms in zip(("dx", "ddt", "dAneg", "dB", "dC", "dh0"), got, want,
                                 (n, n, sum(lens), d, d, 1)):
        ref.check(name, a, b, ref.fp32_bar(2 * longest, terms))
        if name in ("dx", "ddt", "dB", "dC"):
            assert not a[sum(lens):].any(), name


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens", list(LENS))
def test_scan_lengths(lens, dtype):
    check_scan(LENS[lens], 3, 40, 16, dtype, carried=True)


@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 13, 16, 17, 24, 32, 33, 64])
def test_scan_states(n):
    check_scan(LENS["mixed"], 0, 33, n, F32, carried=True)
    check_scan([70, 2], 1, 17, n, BF16, carried=False)


@pytest.mark.parametrize("d", [1, 15, 16, 64, 65, 200])
def test_scan_widths(d):
    check_scan(LENS["two_long"], 5, d, 16, F32, carried=False, cu_dtype=torch.int64)


def test_scan_many_sequences():
    """More sequences than one round of the search probes."""
    lens = [(i * 7) % 5 for i in range(700)]
    check_scan(lens, 2, 20, 16, F32, carried=True)


def test_scan_without_state_or_gradient():
    ts = scan_inputs(LENS["mixed"], 0, 24, 16, F32, False, False)
    y = selective_scan_packed(*ts[:5], _cu(LENS["mixed"]))
    y2, _ = selective_scan_packed(*ts[:5], _cu(LENS["mixed"]), return_state=True)
    assert torch.equal(y, y2)
    # a gradient of the state alone
    x = ts[0].clone().requires_grad_(True)
    _, h = selective_scan_packed(x, *ts[1:5], _cu(LENS["mixed"]), return_state=True)
    (dx,) = torch.autograd.grad(h.sum(), [x])
    xr = _d(x)
    _, hr = ref.scan(xr, *(_d(t) for t in ts[1:5]), LENS["mixed"], None)
    (want,) = torch.autograd.grad(hr.sum(), [xr])
    ref.check("dx", dx, want, ref.fp32_bar(260, 16))


def test_scan_slices_of_wider_tensors():
    """Rows apart, and 16-bit rows at odd addresses."""
    lens = LENS["mixed"]
    for dtype in (F32, BF16):
        x, dt, aneg, b_in, c_in, _ = scan_inputs(lens, 0, 24, 8, dtype, False, False)
        rows = x.shape[0]
        wide = torch.randn(rows, 24 + 24 + 8 + 8 + 1, device="cuda").to(dtype)
        wide[:, 1:25], wide[:, 25:49], wide[:, 49:57], wide[:, 57:] = x, dt, b_in, c_in
        views = wide[:, 1:25], wide[:, 25:49], wide[:, 49:57], wide[:, 57:]
        got = selective_scan_packed(views[0], views[1], aneg, views[2], views[3], _cu(lens))
        assert torch.equal(got, selective_scan_packed(x, dt, aneg, b_in, c_in, _cu(lens)))
        # an expanded and a transposed operand are copied
        got = selective_scan_packed(x[:1].expand(rows, -1), dt.t().contiguous().t(), aneg, b_in,
                                    c_in, _cu(lens))
        want = selective_scan_packed(x[:1].repeat(rows, 1), dt, aneg, b_in, c_in, _cu(lens))
        assert torch.equal(got, want)


def conv_inputs(lens, pad, d, k, dtype, wdtype, carried, grad, seed=0):
    g = torch.Generator().manual_seed(seed)
    rows = sum(lens) + pad
    x = torch.randn(rows, d, generator=g).to(dtype)
    w = torch.randn(d, 1, k, generator=g).to(wdtype)
    bias = torch.randn(d, generator=g).to(wdtype)
    win = torch.randn(len(lens), d, k - 1, generator=g).to(dtype) if carried else None
    return [_leaf(t, grad) for t in (x, w, bias)] + [_leaf(win, grad) if carried else None]


def check_conv(lens, pad, d, k, dtype, wdtype, carried, seed=0):
    ts = conv_inputs(lens, pad, d, k, dtype, wdtype, carried, True, seed)
    out, win = conv1d_silu_packed(*ts[:3], _cu(lens), window=ts[3], return_window=True)
    rs = [_d(t) for t in ts]
    outr, winr = ref.conv(rs[0], rs[1].view(d, k), rs[2], lens, rs[3])
    bar = ref.U * (4 * k + 24)
    ref.check("out", out, outr.detach(), bar)
    assert torch.equal(win.detach().double().cpu(), winr.detach())   # inputs, as they are
    assert not out[sum(lens):].any()
    if not sum(lens):
        return
    g = torch.Generator().manual_seed(seed + 1)
    dout, dwin = (torch.randn(t.shape, generator=g).to(dtype) for t in (out, win))
    outs, ups, outsr = [out, win], [dout, dwin], [outr, winr]
    if k == 1:
        outs, ups, outsr = outs[:1], ups[:1], outsr[:1]
    leaves = [t for t in ts if t is not None and t.numel()]
    got = torch.autograd.grad(outs, leaves, [t.cuda() for t in ups])
    want = torch.autograd.grad(outsr, [t for t in rs if t is not None and t.numel()],
                               [t.double() for t in ups])
    for name, a, b, terms in zip(("dx", "dw", "dbias", "dwindow"), got, want,
                                 (k * k, sum(lens), sum(lens), k * k)):
        ref.check(name, a, b, bar + ref.U * 8 * terms ** 0.5)
    assert not got[0][sum(lens):].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens", list(LENS))
def test_conv_lengths(lens, dtype):
    check_conv(LENS[lens], 3, 40, 4, dtype, dtype, carried=True)


@pytest.mark.parametrize("k", [1, 2, 3, 5, 6, 7, 8])
def test_conv_taps(k):
    check_conv(LENS["mixed"], 0, 33, k, F32, F32, carried=True)
    check_conv(LENS["mixed"], 1, 64, k, BF16, F32, carried=True)
    check_conv(LENS["mixed"], 1, 24, k, F16, F16, carried=False)


@pytest.mark.parametrize("d", [1, 8, 257, 520, 1030])
def test_conv_widths(d):
    check_conv(LENS["two_long"], 2, d, 4, BF16, BF16, carried=False)


def test_conv_half_of_in_proj():
    for dtype in (F32, BF16):
        for d, off in ((64, 0), (64, 64), (33, 33)):
            xz = torch.randn(236, 2 * 64, device="cuda").to(dtype)
            w = torch.randn(d, 4, device="cuda").to(dtype)
            b = torch.randn(d, device="cuda").to(dtype)
            x = xz[:, off:off + d]
            cu = _cu(LENS["mixed"])
            got = conv1d_silu_packed(x, w, b, cu)
            assert torch.equal(got, conv1d_silu_packed(x.contiguous(), w, b, cu))
            x = x.detach().requires_grad_(True)
            g = torch.randn(236, 2 * 64, device="cuda").to(dtype)[:, off:off + d]
            (dx,) = torch.autograd.grad(conv1d_silu_packed(x, w, b, cu), [x], [g])
            xc = x.detach().contiguous().requires_grad_(True)
            (want,) = torch.autograd.grad(conv1d_silu_packed(xc, w, b, cu), [xc], [g.contiguous()])
            assert torch.equal(dx, want)
