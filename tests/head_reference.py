"""The head's losses in 64 bits, and how far a kernel's results may be off.

Bounds, per element, from the operands' magnitudes (all in 64 bits). The products
are exact (16-bit operands) or those of three bf16 parts, and a sum of K terms
adds 16 of them at a time to an fp32 running sum, which rounds or truncates by at
most 2^-23 of a magnitude that sum |a_k b_k| bounds; fp32 takes six such additions
per 16 terms and 40 for its parts, splits and ends, so with m = sum |a_k b_k|
  sum:      (6 K / 16 + 40) 2^-23 m
  log-sum-exp: the largest error of its logits; the exponents' rounding (half a
            unit of |y| <= 64 at the terms that count, 2^-19), the exponential's
            and the logarithm's own (2^-21), up to 100 additions in a row
            (100 2^-24): 2^-17 in all, and 2^-22 of its own size
  p:        its logit's and the log-sum-exp's error, relative to p; the
            exponential instruction gives 0 below 2^-126, the smallest normal
  q:        the exponent (v - max v) log2(e) / t has four roundings (the constant,
            the division, the difference, the product), each half a unit of it:
            2^-22 (max v - v) / t relative, and 2^-20 for the exponential, the sum
            and the division
  dz:       p's error, and for 16-bit operands the rounding to them, half a
            unit: eps / 2 relative
  dh, dW:   dz's error times |W| or |h|, the sum's, and the result's own
            rounding (eps / 2 relative, or half of the smallest subnormal)
"""
from __future__ import annotations

import math

import torch

UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def sum_error(k: int) -> float:
    return (6 * k / 16 + 40) * 2.0 ** -23


def _lse_error(zerr: torch.Tensor, lse: torch.Tensor) -> torch.Tensor:
    worst = zerr.amax(1) if zerr.shape[1] else zerr.new_zeros(len(zerr))
    return worst + 2.0 ** -17 + 2.0 ** -22 * lse.abs()


def teacher(values, ids, temperature):
    """(q, log q, q's relative error, counted) of the teacher's words, in 64 bits."""
    y = (values.double() / temperature).masked_fill(ids < 0, -math.inf)
    top = y.amax(1, keepdim=True)
    counted = top[:, 0] != -math.inf
    lse = torch.logsumexp(y, 1, keepdim=True)
    logq = torch.where(counted[:, None], y - lse, -math.inf)
    err = 2.0 ** -20 + 2.0 ** -22 * torch.where(y > -math.inf, top - y, 0.0)
    return logq.exp(), logq, err, counted


class Reference:
    """Losses, their gradient to the logits per unit of upstream, and the errors
    that are allowed them, for logits z (R, V) in 64 bits whose own error is
    zerr. targets (R) or a teacher (values, ids, temperature)."""

    def __init__(self, z, zerr, targets=None, ignore=-100, words=None, unit=0.0):
        rows, vocab = z.shape
        t = 1.0 if words is None else words[2]
        y, yerr = z / t, zerr / t
        lse = torch.logsumexp(y, 1)
        lse_err = _lse_error(yerr, lse)
        p = (y - lse[:, None]).exp()
        at = torch.arange(rows, device=z.device)
        dz = p.clone()
        if words is None:
            self.counted = targets != ignore
            id_ = torch.where(self.counted, targets, 0)
            self.loss = torch.where(self.counted, lse - z[at, id_], 0.0)
            self.loss_err = torch.where(self.counted, lse_err + zerr[at, id_]
                                        + 2.0 ** -22 * z[at, id_].abs(), 0.0)
            dz[at, id_] -= 1.0
        else:
            values, ids, _ = words
            q, logq, qerr, self.counted = teacher(values, ids, t)
            w = ids.clamp(min=0)
            parts = torch.where(q > 0, q * (logq - y.gather(1, w) + lse[:, None]), 0.0)
            mag = torch.where(q > 0, q * (logq.abs() + y.gather(1, w).abs()
                                          + lse.abs()[:, None]), 0.0)
            self.loss = torch.where(self.counted, t * t * parts.sum(1), 0.0)
            self.loss_err = torch.where(
                self.counted, t * t * (lse_err + (q * yerr.gather(1, w)).sum(1)
                                       + ((qerr + 2.0 ** -20) * mag).sum(1)), 0.0)
            dz.scatter_add_(1, w, -q)
        self.dz = torch.where(self.counted[:, None], t * dz, 0.0)
        perr = p * (yerr + lse_err[:, None] + 2.0 ** -20) + 2.0 ** -126
        if words is not None:
            perr.scatter_add_(1, w, qerr * q)
        self.dz_err = torch.where(self.counted[:, None], t * perr, 0.0) + unit * self.dz.abs()

    def reduced(self, reduction):
        """(loss, its allowed error, the factor on each row's gradient)."""
        n = self.counted.sum()
        if reduction == "none":
            return self.loss, self.loss_err, 1.0
        share = n.double() if reduction == "mean" else 1.0
        loss = self.loss.sum() / share
        return loss, self.loss_err.sum() / share + 2.0 ** -23 * loss.abs(), 1.0 / share


def assert_within(name, got, want, err):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bad = ~((got - want).abs() <= err)
    if bad.any():
        i = int(((got - want).abs() - err).nan_to_num(nan=math.inf).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} elements off; worst at "
                             f"{i}: {got.flatten()[i]:.9g} for {want.flatten()[i]:.9g}, allowed "
                             f"{(err + torch.zeros_like(want)).flatten()[i]:.3g}")


def assert_head(name, got, h, w, upstream, reduction, dtype, **kind):
    """got = (loss, dh, dW) against the reference on h (R, D), w (V, D)."""
    hd, wd = h.double(), w.double()
    k = h.shape[1]
    z = hd @ wd.t()
    zerr = sum_error(k) * (hd.abs() @ wd.abs().t())
    unit = UNIT[dtype]
    ref = Reference(z, zerr, unit=unit, **kind)
    loss, err, share = ref.reduced(reduction)
    assert_within(name + " loss", got[0], loss, err + 1e-30)
    up = upstream.double() * share
    up = (up[:, None] if up.dim() else up)
    dz, dz_err = ref.dz * up, ref.dz_err * up.abs() + 2.0 ** -22 * (ref.dz * up).abs()
    if dtype == torch.float16:   # stored scaled so that the largest is near 2^15: the
        dz_err = dz_err + 2.0 ** -25 * up.abs().max() * 2.0 ** -13   # smallest step
    for what, g, a, a_err, b in (("dh", got[1], dz, dz_err, wd),
                                 ("dW", got[2], dz.t(), dz_err.t(), hd)):
        if g is None:
            continue
        want = a @ b
        bound = a_err @ b.abs() + sum_error(a.shape[1]) * (a.abs() @ b.abs())
        bound = bound * (1 + 2 * unit) + max(unit, 2.0 ** -23) * want.abs() + TINY[dtype] + 1e-37
        assert_within(f"{name} {what}", g, want, bound)
