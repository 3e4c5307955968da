"""Distillation of given logits far from zero: rows that a mask of a large finite value,
or the type's lowest, leaves nothing of, and common offsets."""
from __future__ import annotations

import math

import pytest
import torch

from mamba_metal_scan_amd import distill_loss

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (1 << 31))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 17, 300, 20011])
@pytest.mark.parametrize("mask", ["lowest", -1e4, -1e9, -1e30])
def test_rows_of_one_value(vocab, dtype, mask):
    """A row whose logits are all a mask's value or the type's lowest (a mask that
    leaves nothing), or all its highest: the uniform distribution. So with
    some of them -inf: uniform over the others. Of z_v all alike: p = 1 / n, loss =
    sum q ln q + ln n: n terms' sum of ones is exact, and log2, its product with ln 2
    and the teacher's own terms take 2^-20 of magnitudes below 2 ln n + 8; p's
    exponential and quotient 2^-20 relative, and the result's rounding."""
    dt = TYPES[dtype]
    fi = torch.finfo(dt)
    mask = fi.min if mask == "lowest" else max(mask, fi.min)
    k = min(5, vocab)
    g = _gen(vocab)
    values = torch.randn(4, k, generator=g, device=DEV)
    ids = torch.arange(k, device=DEV).expand(4, k).contiguous()
    z = torch.full((4, vocab), mask, dtype=dt, device=DEV)
    z[1] = fi.max
    n = torch.full((4,), float(vocab), dtype=torch.float64, device=DEV)
    if vocab > 10:
        z[2, k + 2:] = -math.inf
        n[2] = k + 2
        z[3, 9:] = -math.inf   # below the lowest: by a word that is not masked
        z[3, :9] = 0.0
        n[3] = 9
    for t in (1.0, 2.0, 0.5):
        a = z.clone().requires_grad_()
        loss = distill_loss(a, values, ids, temperature=t, reduction="none")
        grad, = torch.autograd.grad(loss, [a], torch.ones_like(loss))
        q = (values.double() / t).softmax(1)
        want = t * t * ((q * q.log()).sum(1) + n.log())
        assert ((loss.double() - want).abs() <= t * t * 2.0 ** -20 * (2 * n.log() + 8)).all(), \
            (loss, want)
        p = torch.where(z == -math.inf, 0.0, 1.0) / n[:, None]
        dz = p.clone()
        dz[:, :k] -= q
        err = t * 2.0 ** -18 * (p + dz.abs()) + fi.eps * t * dz.abs() + 2.0 ** -24
        assert ((grad.double() - t * dz).abs() <= err).all()


@pytest.mark.parametrize("offset", [-1e6, 3e5, 2.0 ** 30])
def test_common_offsets(offset):
    """Logits of an offset that all share: the same distribution (in 64 bits, of the
    logits as they are rounded), to fp32's rounding of differences below 64."""
    g = _gen(7)
    z = 3 * torch.randn(5, 3001, generator=g, device=DEV) + offset
    values = torch.randn(5, 6, generator=g, device=DEV)
    ids = torch.randint(0, 3001, (5, 6), generator=g, device=DEV)
    a = z.clone().requires_grad_()
    loss = distill_loss(a, values, ids, temperature=2.0, reduction="none")
    grad, = torch.autograd.grad(loss, [a], torch.ones_like(loss))
    logp = (z.double() / 2).log_softmax(1)
    q = (values.double() / 2).softmax(1)
    want = 4 * (q * (q.log() - logp.gather(1, ids))).sum(1)
    # each of the exponents, the 3001 sums' rounding (3001 2^-24 at most) and the rest
    assert ((loss.double() - want).abs() <= 4 * (2.0 ** -18 * 64 + 2.0 ** -12)).all()
    dz = logp.exp()
    p = 2 * dz
    dz = 2 * dz.scatter_add_(1, ids, -q)
    assert ((grad.double() - dz).abs() <= (2.0 ** -18 * 64 + 2.0 ** -12) * p
            + 2.0 ** -18 * dz.abs() + 2.0 ** -120).all()


def test_rows_of_the_lowest_value_beside_others():
    """Such rows change nothing in the rows beside them, and a row of -inf alone has
    no distribution: NaN, as the logits' softmax."""
    g = _gen(5)
    z = 3 * torch.randn(6, 3001, generator=g, device=DEV)
    values = torch.randn(6, 4, generator=g, device=DEV)
    ids = torch.randint(0, 3001, (6, 4), generator=g, device=DEV)
    want = distill_loss(z, values, ids, reduction="none")
    masked = z.clone()
    masked[1] = torch.finfo(torch.float32).min
    masked[4] = -math.inf
    a = masked.requires_grad_()
    loss = distill_loss(a, values, ids, reduction="none")
    grad, = torch.autograd.grad(loss, [a], torch.ones_like(loss))
    rest = [0, 2, 3, 5]
    assert torch.equal(loss[rest], want[rest])
    assert torch.isfinite(loss[1]) and torch.isfinite(grad[1]).all()
    assert torch.isnan(loss[4]) and torch.isnan(grad[4]).all()


@pytest.mark.parametrize("temperature", [1e-29, 1e-25, 1e-20, 1e-10, 1e-3, 1e2, 1e6, 1e12, 1e18])
def test_any_temperature(temperature):
    """From one word that has all the weight to the uniform distribution. The loss is a
    sum of terms of one sign here (k of 3001 words), each of a few roundings and the
    log-sum-exp's of 3001 2^-24 at most."""
    g = _gen(11)
    z = 3 * torch.randn(5, 3001, generator=g, device=DEV)
    values = torch.randn(5, 6, generator=g, device=DEV)
    ids = torch.randint(0, 3001, (5, 6), generator=g, device=DEV)
    a = z.clone().requires_grad_()
    t = float(torch.tensor(temperature))   # as the kernel has it
    loss = distill_loss(a, values, ids, temperature=temperature, reduction="none")
    grad, = torch.autograd.grad(loss, [a], torch.ones_like(loss))
    logp = (z.double() / t).log_softmax(1)
    q = (values.double() / t).softmax(1)
    terms = torch.where(q > 0, q * ((values.double() / t).log_softmax(1) - logp.gather(1, ids)), 0.0)
    want = t * t * terms.sum(1)
    assert ((loss.double() - want).abs() <= 2.0 ** -12 * want.abs()).all(), (loss, want)
    dz = (t * logp.exp())
    err = 2.0 ** -12 * dz
    dz.scatter_add_(1, ids, -t * q)
    assert ((grad.double() - dz).abs() <= err + 2.0 ** -18 * dz.abs() + t * 2.0 ** -100).all()
