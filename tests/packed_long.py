"""The packed scan and its gradients in 64 bits for long sequences, on whatever device its inputs
are: the recurrences along time by doubling, some channels at a time."""
from __future__ import annotations

import torch

from packed_reference import spans


def _along(a, b, first):
    """h_t = a_t h_{t-1} + b_t from h_{-1} = first, t along dim 0."""
    b = b.clone()
    b[0] += a[0] * first
    a, step = a.clone(), 1
    while step < a.shape[0]:
        b[step:] += a[step:] * b[:-step]      # (the right side is formed first)
        a[step:] = a[step:] * a[:-step]
        step *= 2
    return b


def scan(x, dt, aneg, b_in, c_in, lens, h0, dy, dh):
    """[y, h_last, dx, ddt, dAneg, dB, dC, dh0], float64 of float64."""
    n = aneg.shape[1]
    y, dx, ddt = (torch.zeros_like(x) for _ in range(3))
    db, dc = torch.zeros_like(b_in), torch.zeros_like(c_in)
    h_last, dh0, da = h0.clone(), dh.clone(), torch.zeros_like(aneg)
    for s, (lo, hi) in enumerate(spans(lens)):
        if lo == hi:
            continue
        width = max(1, (1 << 25) // ((hi - lo) * n))
        for d0 in range(0, x.shape[1], width):
            ch = slice(d0, d0 + width)
            xs, ds, up = (t[lo:hi, ch, None] for t in (x, dt, dy))
            bs, cs = b_in[lo:hi, None], c_in[lo:hi, None]
            decay = torch.exp(-ds * aneg[ch])
            h = _along(decay, ds * xs * bs, h0[s, ch])
            y[lo:hi, ch] = (h * cs).sum(-1)
            h_last[s, ch] = h[-1]
            # g_t = dy_t C_t + decay_{t+1} g_{t+1}, the last with dh
            after = torch.cat([decay[1:], torch.ones_like(decay[:1])])
            g = _along(after.flip(0), (up * cs).flip(0), dh[s, ch]).flip(0)
            through = decay * g                                   # to h_{t-1}
            q = through * torch.cat([h0[s, ch][None], h[:-1]])
            gb = (g * bs).sum(-1)
            dx[lo:hi, ch] = gb * ds[..., 0]
            ddt[lo:hi, ch] = gb * xs[..., 0] - (q * aneg[ch]).sum(-1)
            da[ch] -= (q * ds).sum(0)
            db[lo:hi] += (g * ds * xs).sum(1)
            dc[lo:hi] += (h * up).sum(1)
            dh0[s, ch] = through[0]
    return [y, h_last, dx, ddt, da, db, dc, dh0]
