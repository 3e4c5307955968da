"""The packed operators, slot steps and sampling where calls can go wrong: captured graphs whose
lengths change, streams, repeated calls, offsets past 2^31, numbers in cu_seqlens that do not
hold, refusals, tracing, gradients against differences."""
from __future__ import annotations

import pytest
import torch

import packed_reference as ref
from helpers import assert_close
from mamba_metal_scan_amd import (conv1d_silu_packed, conv1d_silu_step, sample_tokens,
                                  selective_scan_packed, selective_state_step_slots)
from mamba_metal_scan_amd._native import HipScanError

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _cu(lens, dtype=torch.int32):
    return torch.tensor([0] + lens, device="cuda").cumsum(0).to(dtype)


def _scan(rows, d, n, dtype=F32, seed=0, grad=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    ts = [randn(rows, d).to(dtype), (0.001 + 0.1 * torch.sigmoid(randn(rows, d))).to(dtype),
          randn(d, n).exp(), randn(rows, n).to(dtype), randn(rows, n).to(dtype)]
    return [t.requires_grad_(grad) for t in ts]


def _conv(rows, d, k, dtype=F32, seed=0, grad=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ts = [torch.randn(rows, d, generator=g, device="cuda"),
          torch.randn(d, 1, k, generator=g, device="cuda"),
          torch.randn(d, generator=g, device="cuda")]
    return [t.to(dtype).requires_grad_(grad) for t in ts]


def _graph(fn):
    """fn() warmed up on another stream and captured."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_captured_prefill_replays_with_other_lengths():
    rows, d, n = 300, 96, 16
    x, dt, aneg, b, c = _scan(rows, d, n, BF16)
    xc, w, bias = _conv(rows, d, 4, BF16)
    h0, win = torch.randn(5, d, n, device="cuda"), torch.randn(5, d, 3, device="cuda").to(BF16)
    cu = _cu([100, 0, 70, 1, 100])

    def run():
        o, w_out = conv1d_silu_packed(xc, w, bias, cu, window=win, return_window=True)
        y, h = selective_scan_packed(o, dt, aneg, b, c, cu, h0=h0, return_state=True)
        return o, w_out, y, h

    graph, outs = _graph(run)
    for i, lens in enumerate(([100, 0, 70, 1, 100], [0, 300, 0, 0, 0], [1, 2, 3, 4, 5],
                              [60, 60, 60, 60, 60], [0, 0, 0, 0, 0])):
        cu.copy_(_cu(lens))
        xc.copy_(torch.randn(rows, d, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, run()):
            assert torch.equal(got, want), (i, lens)
        xc.sum().item()      # the program's own work between the replays


def test_captured_training_step_replays():
    """Forward and backward in one graph, with no eager graph of the leaves alive."""
    lens = [70, 33, 1, 96]
    ts = _scan(200, 64, 16, F32, grad=True)
    cs = _conv(200, 64, 4, F32, grad=True)
    cu, dy = _cu(lens), torch.randn(200, 64, device="cuda")

    def run():
        o = conv1d_silu_packed(*cs, cu)
        y = selective_scan_packed(o, *ts[1:], cu)
        return torch.autograd.grad(y, cs + ts[1:], dy)

    want = [g.clone() for g in run()]
    graph, outs = _graph(run)
    for _ in range(4):
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert torch.equal(got, w)
        dy.sum().item()


def test_captured_token_replays_with_other_slots():
    rows, pool, d, n, vocab = 8, 20, 128, 16, 9000
    x, dt, aneg, b, c = _scan(rows, d, n)
    _, w, bias = _conv(1, d, 4)
    slots = torch.arange(rows, device="cuda", dtype=torch.int32)
    h, win = torch.randn(pool, d, n, device="cuda"), torch.randn(pool, d, 3, device="cuda")
    head, u = torch.randn(d, vocab, device="cuda") / 8, torch.rand(rows, device="cuda")
    k = torch.full((rows,), 0, device="cuda")

    def run():
        o = conv1d_silu_step(x, w, bias, win, slots)
        y = selective_state_step_slots(h, o, dt, aneg, b, c, slots)
        return y, *sample_tokens(y @ head, u, top_k=k, top_p=0.9, return_logprobs=True)

    graph, outs = _graph(run)
    for i in range(5):
        perm = torch.randperm(pool, device="cuda")[:rows].to(torch.int32)
        perm[i] = -1
        slots.copy_(perm)
        k.copy_(torch.randint(0, 60, (rows,), device="cuda"))
        h1, w1 = h.clone(), win.clone()
        graph.replay()
        torch.cuda.synchronize()
        h2, w2 = h.clone(), win.clone()
        got = [o.clone() for o in outs]
        h.copy_(h1)
        win.copy_(w1)
        for a, b_ in zip(got, run()):
            assert torch.equal(a, b_), i
        assert torch.equal(h, h2) and torch.equal(win, w2)


def test_two_streams_at_once():
    """Calls on two streams, their workspaces their own."""
    lens = [700, 900, 448]
    jobs = []
    for seed in (1, 2):
        ts = _scan(2048, 256, 16, BF16, seed=seed, grad=True)
        dy = torch.randn(2048, 256, device="cuda").to(BF16)
        z, u = torch.randn(16, 20000, device="cuda"), torch.rand(16, device="cuda")
        jobs.append((ts, dy, z, u))

    def run(ts, dy, z, u):
        y = selective_scan_packed(*ts, _cu(lens))
        return (*torch.autograd.grad(y, ts, dy), sample_tokens(z, u, top_p=0.9))

    want = [run(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for s, j in zip(streams, jobs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run(*j))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_the_same_bits_every_time():
    lens = [600, 1, 0, 300, 123]
    ts = _scan(1030, 200, 16, BF16, grad=True)
    cs = _conv(1030, 200, 4, BF16, grad=True)
    dy = torch.randn(1030, 200, device="cuda").to(BF16)
    z, u = torch.randn(64, 30000, device="cuda"), torch.rand(64, device="cuda")

    def run():
        y = selective_scan_packed(*ts, _cu(lens))
        o = conv1d_silu_packed(*cs, _cu(lens))
        return (y, o, *torch.autograd.grad([y, o], ts + cs, [dy, dy]),
                *sample_tokens(z, u, top_p=0.8, return_logprobs=True))

    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


def test_offsets_past_2_to_the_31():
    """More than 2^31 elements: the last sequence of a long packed tensor, the last entry of a large
    pool, the last rows of many logits, as of that part alone."""
    rows, d, n, last = 1_060_000, 2048, 16, 300
    assert rows * d > 2 ** 31
    lens = [rows - last, last]
    x = torch.empty(rows, d, device="cuda", dtype=BF16).normal_()
    w, bias = torch.randn(d, 4, device="cuda").to(BF16), torch.randn(d, device="cuda").to(BF16)
    o = conv1d_silu_packed(x, w, bias, _cu(lens))
    tail = x[-last:].contiguous()
    assert torch.equal(o[-last:], conv1d_silu_packed(tail, w, bias, _cu([last])))
    del o
    small = _scan(last, d, n, BF16)
    dt = torch.full_like(x, 0.02)
    b, c = (torch.randn(rows, n, device="cuda").to(BF16) for _ in range(2))
    dt[-last:], b[-last:], c[-last:] = small[1], small[3], small[4]
    y, h = selective_scan_packed(x, dt, small[2], b, c, _cu(lens), return_state=True)
    # (pieces of another length: the same within their rounding)
    yt, ht = selective_scan_packed(tail, *small[1:], _cu([last]), return_state=True)
    ref.check("y", y[-last:], yt.double().cpu(), 2.0 ** -7)
    assert_close("h", h[1], ht[0], 1e-5)
    del x, dt, b, c, y
    pool, d = 35_000, 4096
    assert pool * d * n > 2 ** 31
    hp = torch.zeros(pool, d, n, device="cuda")
    hp[-1].normal_()
    x1, dt1, aneg, b1, c1 = _scan(2, d, n)
    one = hp[-1:].clone()
    at = torch.tensor([3, pool - 1], device="cuda")
    y = selective_state_step_slots(hp, x1, dt1, aneg, b1, c1, at)
    y1 = selective_state_step_slots(one, x1[1:], dt1[1:], aneg, b1[1:], c1[1:])
    assert torch.equal(y[1:], y1) and torch.equal(hp[-1:], one)
    del hp
    rows, vocab = 17_000, 131072
    assert rows * vocab > 2 ** 31
    z = torch.empty(rows, vocab, device="cuda", dtype=BF16).normal_()
    u = torch.rand(rows, device="cuda")
    t = sample_tokens(z, u, top_k=20, temperature=0.7)
    assert torch.equal(t[-5:], sample_tokens(z[-5:].contiguous(), u[-5:], top_k=20,
                                             temperature=0.7))


def test_numbers_that_are_no_lengths_stay_in_bounds():
    """cu_seqlens that do not rise, or go past the rows, give undefined results within the tensors:
    the rows around them keep their bits."""
    rows, d, n = 100, 40, 16
    for cu in ([0, 50, 20, 100], [-5, 50, 200], [90, 10, 95], [0, 1 << 30], [100, 100, 100, 0]):
        for dtype in (torch.int32, torch.int64):
            at = torch.tensor(cu, device="cuda", dtype=dtype)
            ts = _scan(rows, d, n, grad=True)
            y, h = selective_scan_packed(*ts, at, return_state=True)
            torch.autograd.grad(y, ts, torch.ones_like(y))
            cs = _conv(rows, d, 4, grad=True)
            o, _ = conv1d_silu_packed(*cs, at, return_window=True)
            torch.autograd.grad(o, cs, torch.ones_like(o))
    torch.cuda.synchronize()


def test_infinities_and_nan_stay_in_their_sequence():
    lens = [40, 50, 60]
    ts = _scan(150, 32, 16)
    cs = _conv(150, 32, 4)
    y, o = selective_scan_packed(*ts, _cu(lens)), conv1d_silu_packed(*cs, _cu(lens))
    bad = [t.clone() for t in ts]
    bad[0][45], bad[3][60] = float("inf"), float("nan")
    cx = cs[0].clone()
    cx[42] = float("nan")
    y2, o2 = selective_scan_packed(*bad, _cu(lens)), conv1d_silu_packed(cx, *cs[1:], _cu(lens))
    for a, b in ((y, y2), (o, o2)):
        assert torch.equal(a[:40], b[:40]) and torch.equal(a[90:], b[90:])
        assert torch.isnan(b[40:90]).any()
    # and what lies behind the last sequence is not looked at
    bad = [t.clone().requires_grad_(True) for t in ts]
    with torch.no_grad():
        for i in (0, 1, 3, 4):
            bad[i][90:] = float("nan")
    good = [t.clone().requires_grad_(True) for t in ts]
    dy = torch.randn(150, 32, device="cuda")
    got = torch.autograd.grad(selective_scan_packed(*bad, _cu(lens[:2])), bad, dy)
    want = torch.autograd.grad(selective_scan_packed(*good, _cu(lens[:2])), good, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_against_differences():
    """Central differences of the fp32 operators in one random direction per input: a step of
    2^-8 of unit numbers leaves the third derivatives' part, 2^-16 of it, and the outputs'
    rounding, 2^-24 sqrt(sum of squares) / 2^-8."""
    lens = [9, 1, 0, 20]
    g = torch.Generator(device="cuda").manual_seed(4)
    ts = [t.detach() for t in _scan(32, 24, 8)]
    h0 = torch.randn(4, 24, 8, generator=g, device="cuda")
    cs = [t.detach() for t in _conv(32, 24, 4)]
    win = torch.randn(4, 24, 3, generator=g, device="cuda")
    cu = _cu(lens)

    def scan(*a):
        return selective_scan_packed(*a[:5], cu, h0=a[5], return_state=True)

    def conv(*a):
        return conv1d_silu_packed(*a[:3], cu, window=a[3], return_window=True)

    for fn, args in ((scan, ts + [h0]), (conv, cs + [win])):
        leaves = [a.clone().requires_grad_(True) for a in args]
        outs = fn(*leaves)
        ups = [torch.randn(o.shape, generator=g, device="cuda") for o in outs]
        grads = torch.autograd.grad(outs, leaves, ups)
        for i, gr in enumerate(grads):
            way = torch.randn(gr.shape, generator=g, device="cuda")
            if fn is scan and i == 1:
                way *= 0.05            # dt is of that size
            step = 2.0 ** -8
            vals = []
            for sign in (1.0, -1.0):
                moved = [a + sign * step * way if j == i else a for j, a in enumerate(args)]
                vals.append(sum((o.double() * u.double()).sum() for o, u in zip(fn(*moved), ups)))
            diff = float((vals[0] - vals[1]) / (2 * step))
            mine = float((gr.double() * way.double()).sum())
            size = float((gr.double() * way.double()).abs().sum())
            assert abs(diff - mine) <= 2e-3 * size + 2e-3, (fn.__name__, i, diff, mine)


def test_gradients_of_some_inputs_and_odd_gradients():
    lens = [30, 34]
    ts = _scan(64, 48, 16)
    x = ts[0].clone().requires_grad_(True)
    y = selective_scan_packed(x, *ts[1:], _cu(lens))
    dy = torch.randn(48, 64, device="cuda").t()             # another layout
    (a,) = torch.autograd.grad(y, [x], dy)
    y = selective_scan_packed(x, *ts[1:], _cu(lens))
    (b,) = torch.autograd.grad(y, [x], dy.contiguous())
    assert torch.equal(a, b)
    y = selective_scan_packed(x, *ts[1:], _cu(lens))
    (c,) = torch.autograd.grad(y.sum(), [x])                # an expanded gradient
    y = selective_scan_packed(x, *ts[1:], _cu(lens))
    (d,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    assert torch.equal(c, d)
    # one tensor as two inputs
    xx = ts[0].clone().requires_grad_(True)
    bb = ts[3].clone().requires_grad_(True)
    y = selective_scan_packed(xx, ts[1], ts[2], bb, bb, _cu(lens))
    (e,) = torch.autograd.grad(y, [bb], torch.ones_like(y))
    b1, b2 = (ts[3].clone().requires_grad_(True) for _ in range(2))
    y = selective_scan_packed(xx, ts[1], ts[2], b1, b2, _cu(lens))
    f = torch.autograd.grad(y, [b1, b2], torch.ones_like(y))
    assert torch.equal(e, f[0] + f[1])
    # saved tensors that come back in another layout, elsewhere
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        y = selective_scan_packed(x, *ts[1:], _cu(lens))
    (g,) = torch.autograd.grad(y, [x], dy.contiguous())
    assert torch.equal(g, b)
    y = selective_scan_packed(x, *ts[1:], _cu(lens))
    with pytest.raises(HipScanError, match="once differentiable"):
        torch.autograd.grad(y.sum(), [x], create_graph=True)
    cs = _conv(64, 48, 4, grad=True)
    o = conv1d_silu_packed(*cs, _cu(lens))
    with pytest.raises(HipScanError, match="once differentiable"):
        torch.autograd.grad(o.sum(), cs, create_graph=True)


def test_refusals():
    x, dt, aneg, b, c = _scan(20, 16, 8)
    cu = _cu([12, 8])
    for match, call in (
            ("two dimensions", lambda: selective_scan_packed(x[None], dt, aneg, b, c, cu)),
            ("must all be", lambda: selective_scan_packed(x.to(BF16), dt, aneg, b, c, cu)),
            ("must all be", lambda: selective_scan_packed(x.double(), dt.double(), aneg,
                                                          b.double(), c.double(), cu)),
            ("dt must have", lambda: selective_scan_packed(x, dt[:, :8], aneg, b, c, cu)),
            ("B must have", lambda: selective_scan_packed(x, dt, aneg, b[:8], c, cu)),
            ("Aneg must have", lambda: selective_scan_packed(x, dt, aneg[:8], b, c, cu)),
            ("Aneg must be float32", lambda: selective_scan_packed(x, dt, aneg.double(), b, c, cu)),
            ("cu_seqlens", lambda: selective_scan_packed(x, dt, aneg, b, c, cu.float())),
            ("cu_seqlens", lambda: selective_scan_packed(x, dt, aneg, b, c, cu[None])),
            ("cu_seqlens", lambda: selective_scan_packed(x, dt, aneg, b, c, cu[:0])),
            ("h0 must have", lambda: selective_scan_packed(x, dt, aneg, b, c, cu,
                                                           h0=aneg.new_zeros(3, 16, 8))),
            ("h0 must be float32", lambda: selective_scan_packed(
                x, dt, aneg, b, c, cu, h0=aneg.new_zeros(2, 16, 8, dtype=BF16)))):
        with pytest.raises((RuntimeError, ValueError), match=match):
            call()
    wide = torch.rand(16, 65, device="cuda")
    b65 = torch.randn(20, 65, device="cuda")
    with pytest.raises(HipScanError, match="N in"):
        selective_scan_packed(x, dt, wide, b65, b65, cu)
    xc, w, bias = _conv(20, 16, 4)
    win = torch.zeros(2, 16, 3, device="cuda")
    for match, call in (
            ("x must be", lambda: conv1d_silu_packed(xc[0], w, bias, cu)),
            ("weight must be", lambda: conv1d_silu_packed(xc, w[:8], bias, cu)),
            ("weight must be", lambda: conv1d_silu_packed(xc, w.view(16, 2, 2), bias, cu)),
            ("K in", lambda: conv1d_silu_packed(xc, w.repeat(1, 1, 3), bias, cu)),
            ("bias must have", lambda: conv1d_silu_packed(xc, w, bias[:3], cu)),
            ("of x's type", lambda: conv1d_silu_packed(xc, w.to(BF16), bias.to(BF16), cu)),
            ("window must have", lambda: conv1d_silu_packed(xc, w, bias, cu, window=win[:1])),
            ("window must be", lambda: conv1d_silu_packed(xc, w, bias, cu, window=win.to(F16))),
            ("in place", lambda: conv1d_silu_step(xc[:2], w, bias,
                                                  win.transpose(0, 1).contiguous().transpose(0, 1))),
            ("without slots", lambda: conv1d_silu_step(xc[:3], w, bias, win)),
            ("slots must be", lambda: conv1d_silu_step(xc[:2], w, bias, win, cu)),
            ("slots must be", lambda: conv1d_silu_step(xc[:2], w, bias, win, cu[:2].float())),
            ("no_grad", lambda: conv1d_silu_step(xc[:2], w.requires_grad_(True), bias, win))):
        with pytest.raises((RuntimeError, ValueError), match=match):
            call()
    h = torch.zeros(2, 16, 8, device="cuda")
    for match, call in (
            ("in place", lambda: selective_state_step_slots(
                h.transpose(1, 2).contiguous().transpose(1, 2), x[:2], dt[:2], aneg, b[:2], c[:2])),
            ("h must be float32", lambda: selective_state_step_slots(
                h.to(BF16), x[:2], dt[:2], aneg, b[:2], c[:2])),
            ("x must have", lambda: selective_state_step_slots(
                h, x[:2, :8], dt[:2], aneg, b[:2], c[:2])),
            ("slots must be", lambda: selective_state_step_slots(
                h, x[:2], dt[:2], aneg, b[:2], c[:2], cu))):
        with pytest.raises((RuntimeError, ValueError), match=match):
            call()


def test_no_rows_and_no_sequences():
    x, dt, aneg, b, c = _scan(0, 16, 8, grad=True)
    h0 = torch.randn(2, 16, 8, device="cuda", requires_grad=True)
    y, h = selective_scan_packed(x, dt, aneg, b, c, _cu([0, 0]), h0=h0, return_state=True)
    assert y.shape == (0, 16) and torch.equal(h, h0)
    da, dh = torch.autograd.grad(h, [aneg, h0], torch.ones_like(h))
    assert not da.any() and torch.equal(dh, torch.ones_like(dh))
    x, dt, aneg, b, c = _scan(5, 16, 8, grad=True)
    y = selective_scan_packed(x, dt, aneg, b, c, _cu([]))
    assert not y.any()
    assert not any(g.any() for g in torch.autograd.grad(y, [x, dt, aneg, b, c],
                                                        torch.ones_like(y)))
    cs = _conv(5, 16, 4, grad=True)
    o, w = conv1d_silu_packed(*cs, _cu([]), return_window=True)
    assert not o.any() and w.shape == (0, 16, 3)
    assert not any(g.any() for g in torch.autograd.grad(o, cs, torch.ones_like(o)))
    empty = conv1d_silu_step(cs[0].detach()[:0], cs[1].detach(), cs[2].detach(),
                             torch.zeros(0, 16, 3, device="cuda"))
    assert empty.shape == (0, 16)


def test_torch_compile_traces_in_one_graph():
    lens = [20, 44]
    ts = [t.detach() for t in _scan(64, 32, 16)]
    cs = [t.detach() for t in _conv(64, 32, 4)]
    u = torch.rand(64, device="cuda")
    cu = _cu(lens)

    def f(x, w, bias, dt, aneg, b, c):
        o = conv1d_silu_packed(x, w, bias, cu)
        return selective_scan_packed(o, dt, aneg, b, c, cu, return_state=True)

    args = [t.clone().requires_grad_(True) for t in (*cs, *ts[1:])]
    fc = torch.compile(f, backend="aot_eager", fullgraph=True)
    y, h = f(*args)
    want = torch.autograd.grad([y, h], args, [torch.ones_like(y), torch.ones_like(h)])
    yc, hc = fc(*args)
    got = torch.autograd.grad([yc, hc], args, [torch.ones_like(y), torch.ones_like(h)])
    assert torch.equal(y, yc) and torch.equal(h, hc)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    def s(z):
        return sample_tokens(z * 2.0, u, top_k=5, return_logprobs=True)

    z = torch.randn(64, 500, device="cuda")
    for a, b in zip(torch.compile(s, backend="aot_eager", fullgraph=True)(z), s(z)):
        assert torch.equal(a, b)

    def step(x, h, win):
        o = conv1d_silu_step(x, cs[1], cs[2], win)
        return selective_state_step_slots(h, o, ts[1][:4], ts[2], ts[3][:4], ts[4][:4])

    with torch.no_grad():
        pools = [(torch.ones(4, 32, 16, device="cuda"), torch.ones(4, 32, 3, device="cuda"))
                 for _ in range(2)]
        a = step(cs[0][:4], *pools[0])
        b = torch.compile(step, backend="aot_eager", fullgraph=True)(cs[0][:4], *pools[1])
    assert torch.equal(a, b)
    assert all(torch.equal(p, q) for p, q in zip(*pools))
