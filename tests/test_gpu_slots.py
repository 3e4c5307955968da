"""One token by slot on the GPU against 64 bits: pools larger than the batch, padding, slots that
do not hold, types, widths."""
from __future__ import annotations

import pytest
import torch

import packed_reference as ref
from mamba_metal_scan_amd import conv1d_silu_step, selective_state_step_slots

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _slots(rows, pool, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    s = torch.randperm(pool, generator=g)[:rows]
    if rows > 2:
        s[rows // 2] = -1
    return s.to(dtype)


@pytest.mark.parametrize("rows,pool,d,k,dtype,wdtype,slots", [
    (1, 1, 1, 4, F32, F32, torch.int32), (4, 16, 100, 4, F32, F32, torch.int64),
    (9, 9, 257, 3, BF16, BF16, torch.int32), (300, 301, 64, 8, BF16, F32, torch.int32),
    (7, 20, 33, 2, F16, F16, torch.int64), (5, 6, 40, 1, F32, F32, torch.int32),
    (6, 8, 48, 5, F16, F32, None), (3, 3, 512, 4, BF16, BF16, None)])
def test_conv_step(rows, pool, d, k, dtype, wdtype, slots):
    g = torch.Generator().manual_seed(3)
    x, win = torch.randn(rows, d, generator=g).to(dtype), \
        torch.randn(pool, d, k - 1, generator=g).to(dtype)
    w, b = torch.randn(d, 1, k, generator=g).to(wdtype), torch.randn(d, generator=g).to(wdtype)
    at = _slots(rows, pool, slots, 4) if slots is not None else None
    wide = torch.randn(rows, 2 * d, generator=g).to(dtype).cuda()
    wide[:, d:] = x.cuda()
    pool_t = win.clone().cuda()
    out = conv1d_silu_step(wide[:, d:], w.cuda(), b.cuda(), pool_t,
                           at.cuda() if at is not None else None)
    want_pool, want = win.double(), torch.zeros(rows, d, dtype=torch.float64)
    for r in range(rows):
        s = r if at is None else int(at[r])
        if s < 0:
            continue
        full = torch.cat([want_pool[s], x[r].double()[:, None]], 1)
        pre = b.double() + (full * w.double().view(d, k)).sum(1)
        want[r] = pre * torch.sigmoid(pre)
        want_pool[s] = full[:, 1:]
    ref.check("out", out, want, ref.U * (4 * k + 24))
    assert torch.equal(pool_t.cpu().double(), want_pool)


@pytest.mark.parametrize("rows,pool,d,n,dtype,slots", [
    (1, 1, 1, 1, F32, torch.int32), (4, 16, 100, 16, F32, torch.int64),
    (9, 9, 257, 16, BF16, torch.int32), (300, 301, 64, 8, BF16, torch.int32),
    (7, 20, 33, 3, F16, torch.int64), (5, 6, 40, 64, F32, torch.int32), (6, 8, 48, 24, F16, None),
    (3, 3, 130, 32, BF16, None), (2, 2, 65, 4, F32, None), (2, 5, 7, 13, BF16, torch.int32)])
def test_state_step(rows, pool, d, n, dtype, slots):
    g = torch.Generator().manual_seed(5)
    x, b_in, c_in = (torch.randn(rows, w, generator=g).to(dtype) for w in (d, n, n))
    dt = (0.001 + 0.1 * torch.rand(rows, d, generator=g)).to(dtype)
    aneg = torch.rand(d, n, generator=g) * n
    h = torch.randn(pool, d, n, generator=g)
    at = _slots(rows, pool, slots, 6) if slots is not None else None
    pool_t = h.clone().cuda()
    wide = torch.randn(rows, 3 * d + 1, generator=g).to(dtype).cuda()
    wide[:, 1:d + 1], wide[:, d + 1:2 * d + 1] = x.cuda(), dt.cuda()
    y = selective_state_step_slots(pool_t, wide[:, 1:d + 1], wide[:, d + 1:2 * d + 1], aneg.cuda(),
                                   b_in.cuda(), c_in.cuda(), at.cuda() if at is not None else None)
    want_pool, want = h.double(), torch.zeros(rows, d, dtype=torch.float64)
    for r in range(rows):
        s = r if at is None else int(at[r])
        if s < 0:
            continue
        dd = dt[r].double()[:, None]
        want_pool[s] = (torch.exp(-dd * aneg.double()) * want_pool[s]
                        + dd * x[r].double()[:, None] * b_in[r].double())
        want[r] = want_pool[s] @ c_in[r].double()
    bar = ref.fp32_bar(1, n)
    ref.check("y", y, want, bar)
    ref.check("h", pool_t, want_pool, bar)


def test_slots_that_do_not_hold():
    """Past the pool, or an earlier row's: a row of NaN, no entry touched."""
    d, n, k = 70, 16, 4
    slots = torch.tensor([2, 5, 2, -1, -7, 1, 5, 2, 2**31 - 1], dtype=torch.int64, device="cuda")
    good = [0, 5]          # 2 and 1; 5 is past the pool of 5
    g = torch.Generator().manual_seed(8)
    rows = len(slots)
    x, dt = torch.randn(rows, d, generator=g).cuda(), torch.rand(rows, d, generator=g).cuda()
    b_in, c_in = (torch.randn(rows, n, generator=g).cuda() for _ in range(2))
    aneg, h = torch.rand(d, n, generator=g).cuda(), torch.randn(5, d, n, generator=g).cuda()
    w, b = torch.randn(d, k, generator=g).cuda(), torch.randn(d, generator=g).cuda()
    win = torch.randn(5, d, k - 1, generator=g).cuda()
    for slots_t in (slots, slots.to(torch.int32)):
        h1, h2, w1, w2 = h.clone(), h.clone(), win.clone(), win.clone()
        y = selective_state_step_slots(h1, x, dt, aneg, b_in, c_in, slots_t)
        o = conv1d_silu_step(x, w, b, w1, slots_t)
        yg = selective_state_step_slots(h2, x[good], dt[good], aneg, b_in[good], c_in[good],
                                        slots_t[good])
        og = conv1d_silu_step(x[good], w, b, w2, slots_t[good])
        assert torch.equal(h1, h2) and torch.equal(w1, w2)
        for out, ok in ((y, yg), (o, og)):
            assert torch.equal(out[good], ok)
            assert not out[3:5].any()
            assert torch.isnan(out[[1, 2, 6, 7, 8]]).all()
