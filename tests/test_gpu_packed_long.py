"""The packed scan and conv at the sizes that training has, where a piece is longer than a
sub-chunk and a sequence has many pieces, against 64 bits.

Tolerances are packed_reference's. There a state's error grows by 8 u a row for as long as the
state is remembered. Here dt Aneg is at least 0.02 x 0.2: what a row adds has decayed by
exp(-0.004 m) after m rows, and the sum over all rows before is at most 1 / (1 - exp(-0.004)) < 251
rows' errors, whatever the length. A piece's carry is one exponential of a sum of up to 1024 dt
in place of as many: off by the sum's rounding, below u a row, times x = Aneg sum dt, of a value
that has decayed by exp(-x): x exp(-x) < 1, so within the rows' own."""
from __future__ import annotations

import pytest
import torch

import packed_long
import packed_reference as ref
from mamba_metal_scan_amd import _native, conv1d_silu_packed, selective_scan_packed

F32, BF16 = torch.float32, torch.bfloat16
MEMORY = 251
NAMES = ("y", "h_last", "dx", "ddt", "dAneg", "dB", "dC", "dh0")


def _inputs(lens, pad, d, n, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=device)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=device)

    rows = sum(lens) + pad
    ts = [randn(rows, d).to(dtype), (0.0201 + 0.1 * rand(rows, d)).to(dtype),
          0.2 + n * rand(d, n) ** 2, randn(rows, n).to(dtype), randn(rows, n).to(dtype)]
    return (ts, randn(len(lens), d, n), randn(rows, d).to(dtype), randn(len(lens), d, n))


def test_the_reference_against_autograd():
    lens = [1, 37, 0, 20]
    ts, h0, dy, dh = _inputs(lens, 2, 5, 3, torch.float64, "cpu")
    ts, h0, dh = [t.double() for t in ts], h0.double(), dh.double()
    got = packed_long.scan(*ts, lens, h0, dy, dh)
    leaves = [t.requires_grad_(True) for t in (*ts, h0)]
    y, h = ref.scan(*leaves[:5], lens, leaves[5])
    grads = torch.autograd.grad([y, h], leaves, [dy, dh])
    for name, a, b in zip(NAMES, got, (y, h, *grads)):
        assert torch.allclose(a, b, rtol=1e-11, atol=1e-11), name


def _piece_rows(seqs, rows, d, n, back):
    """Rows of a piece (sixteens) by the workspace, which holds the states of rows // tc + seqs + 1
    pieces."""
    lib = _native.library()
    nbytes = lib.mhs_packed_scan_workspace_bytes(seqs, rows, d, n, back)
    waves = 1 if n <= 16 else 2 if n <= 32 else 4
    if back:
        chans = 32 * (4 // waves)
        nbytes -= 4 * ((d + chans - 1) // chans) * rows * 2 * n
    each = 4 * ((3 if back else 2) * d * n + d)
    assert nbytes % each == 0
    return rows // (nbytes // each - seqs - 1) // 16 * 16


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d,n,dtype", [(8192, 1536, 16, F32), (8192, 1536, 16, BF16),
                                            (4096, 2048, 64, F32), (4096, 2048, 64, BF16),
                                            (6000, 2560, 32, BF16), (32768, 2048, 16, BF16)])
def test_scan_of_many_long_pieces(rows, d, n, dtype):
    """Sequences from rows that no power of two divides, that end 1, 15 and 17 rows into a piece of
    either direction."""
    lens = []
    for tc in (_piece_rows(9, rows, d, n, b) for b in (0, 1)):
        assert tc >= 32, "pieces of one sub-chunk: choose larger sizes"
        lens += [5, 3 * tc + 1, 2 * tc + 15, 4 * tc + 17]
    lens.append(rows - 3 - sum(lens))
    assert lens[-1] > 0 and len(lens) == 9
    ts, h0, dy, dh = _inputs(lens, 3, d, n, dtype, "cuda")
    leaves = [t.requires_grad_(True) for t in (*ts, h0)]
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
    y, h = selective_scan_packed(*leaves[:5], cu, h0=leaves[5], return_state=True)
    grads = torch.autograd.grad([y, h], leaves, [dy, dh])
    want = packed_long.scan(*(t.detach().double() for t in ts), lens, h0.detach().double(),
                            dy.double(), dh.double())
    sizes = dict(y=n, h_last=1, dx=n, ddt=n, dAneg=rows, dB=d, dC=d, dh0=1)
    for name, a, b in zip(NAMES, (y, h, *grads), want):
        passes = 1 if name in ("y", "h_last") else 2
        ref.check(name, a, b.cpu(), ref.fp32_bar(passes * MEMORY, sizes[name]))
    with torch.no_grad():
        y2, h2 = selective_scan_packed(*ts, cu, h0=h0, return_state=True)
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_conv_of_a_training_batch(dtype):
    """8192 x 1536 in 24 documents, the left half of wider rows: against 64 bits, and the same bits
    every time, other calls between them."""
    rows, d, k = 8192, 1536, 4
    g = torch.Generator(device="cuda").manual_seed(2)
    lens = [(i * 97) % 683 for i in range(23)]
    lens.append(rows - sum(lens))
    x = torch.randn(rows, 2 * d, generator=g, device="cuda").to(dtype)[:, :d]
    w = (torch.rand(d, 1, k, generator=g, device="cuda") - 0.5).to(dtype)
    bias = (torch.rand(d, generator=g, device="cuda") - 0.5).to(dtype)
    dout = torch.randn(rows, d, generator=g, device="cuda").to(dtype)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, bias)]

    def run(up):
        out = conv1d_silu_packed(*leaves, cu)
        return [out.detach(), *torch.autograd.grad(out, leaves, up)]

    got = run(dout)
    for _ in range(4):
        run(dout.flip(0))
        assert all(torch.equal(a, b) for a, b in zip(run(dout), got))
    rs = [t.detach().double().requires_grad_(True) for t in leaves]
    out, _ = ref.conv(rs[0], rs[1].view(d, k), rs[2], lens, None)
    want = [out.detach(), *torch.autograd.grad(out, rs, dout.double())]
    bar = ref.U * (4 * k + 24)
    for name, a, b, terms in zip(("out", "dx", "dw", "dbias"), got, want, (0, k * k, rows, rows)):
        ref.check(name, a, b.cpu(), bar + ref.U * 8 * terms ** 0.5)
