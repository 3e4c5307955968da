"""The operators over packed sequences, tokens by slot and sampling in 64 bits on the CPU, from
their definitions, and how far the kernels may be from them.

Tolerances. A result in type t is rounded once: off by at most eps(t) / 2 of its value. Before
that it is computed in fp32, u = 2^-24 being a rounding. A conv's output takes K + 1 roundings of a
sum of K + 1 terms and a few in the sigmoid (hardware exponential and reciprocal: 1 ulp each).
The scan multiplies a state by exp(-dt Aneg) each row, off by (|dt Aneg| + 3) u of its value,
and adds with one rounding: what a state has from m rows before is off by at most m (|dt
Aneg| + 4) u, which with |dt Aneg| <= 4 makes 8 u a row, and no state remembers more rows than
its sequence has. y and the gradients add a fixed-order sum of n terms, n u of the terms'
sizes at most. fp32_bar gives these together, relative to the largest value of the result; for sums
over n random terms that value is about sqrt(n) of theirs.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

U = 2.0 ** -24


def fp32_bar(rows: int, terms: int) -> float:
    """Of results that rows recurrent rows and a sum of `terms` terms go into."""
    return U * (8 * rows + 4 * math.sqrt(terms) + 16)


def check(name, got, ref, bar: float) -> None:
    """got against ref (64 bits): a rounding to got's type, and bar of ref's largest value."""
    assert tuple(got.shape) == tuple(ref.shape), (name, got.shape, ref.shape)
    g = got.detach().double().cpu()
    if g.numel() == 0:
        return
    eps = torch.finfo(got.dtype).eps
    top = ref.abs().max()
    allowed = (0.5 * eps) * ref.abs() + bar * max(float(top), 1e-30)
    if got.dtype == torch.float16:
        allowed = allowed + 2.0 ** -25     # half a step of the smallest halves
    over = ((g - ref).abs() - allowed).max()
    assert not torch.isnan(g).any(), f"{name}: NaN"
    assert over <= 0, f"{name}: off by {float((g - ref).abs().max()):.3e}, largest {float(top):.3e}"


def spans(lens):
    at = 0
    for n in lens:
        yield at, at + n
        at += n


def conv(x, w, bias, lens, window):
    """(out, windows) of x (L, D), w (D, K), window (S, D, K - 1) or None, all float64."""
    d, k = w.shape
    out = torch.zeros_like(x)
    ends = []
    parts = []
    for s, (b, e) in enumerate(spans(lens)):
        before = window[s] if window is not None else x.new_zeros(d, k - 1)
        row = torch.cat([before, x[b:e].t()], 1)
        ends.append(row[:, row.shape[1] - (k - 1):])
        if e > b:
            pre = bias[:, None] + sum(w[:, j:j + 1] * row[:, j:j + e - b] for j in range(k))
            parts.append((pre * torch.sigmoid(pre)).t())
    parts.append(out[sum(lens):])
    return torch.cat(parts), (torch.stack(ends) if ends else x.new_zeros(0, d, k - 1))


def scan(x, dt, aneg, b_in, c_in, lens, h0):
    """(y, states) of the packed scan, float64."""
    ys, hs = [], []
    for s, (b, e) in enumerate(spans(lens)):
        h = h0[s] if h0 is not None else x.new_zeros(aneg.shape)
        for t in range(b, e):
            h = torch.exp(-dt[t][:, None] * aneg) * h + (dt[t] * x[t])[:, None] * b_in[t]
            ys.append(h @ c_in[t])
        hs.append(h)
    y = torch.stack(ys) if ys else x.new_zeros(0, x.shape[1])
    return (torch.cat([y, x.new_zeros(x.shape[0] - y.shape[0], x.shape[1])]),
            torch.stack(hs) if hs else x.new_zeros(0, *aneg.shape))


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability) of one row (float64 list or tensor), word by word."""
    row = [(-math.inf if math.isnan(v) else v) for v in row.tolist()]
    top = max(row)
    if top == -math.inf or not (0 <= temperature < math.inf) or not min_p <= 1 or math.isnan(top_p):
        return -1, math.nan
    order = sorted(range(len(row)), key=lambda i: (-row[i], i))
    if temperature == 0:
        return order[0], 0.0
    w = {i: (1.0 if row[i] == top else
             0.0 if top == math.inf else math.exp((row[i] - top) / temperature)) for i in order}
    # sums without rounding: integers of 2^-200 (the fp32 settings are whole ones of 2^-149 or more)
    n = {i: int(Fraction(v) * 2 ** 200) for i, v in w.items()}
    if 0 < top_k < len(order):
        order = order[:top_k]
    if top_p < 1:
        border, run, kept = Fraction(top_p) * sum(n[i] for i in order), 0, []
        for i in order:
            if kept and not run < border:
                break
            kept.append(i)
            run += n[i]
        order = kept
    order = sorted(i for i in order if w[i] >= min_p)
    total = sum(n[i] for i in order)
    border, run, token = Fraction(u) * total, 0, None
    for i in order:
        run += n[i]
        if n[i]:
            token = i
            if run > border:
                break
    return token, math.log(n[token] / total)
