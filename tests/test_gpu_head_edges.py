"""The head's losses at the edges of what their contract allows: infinities and NaN in
the weight beside rows that do not count."""
from __future__ import annotations

import math

import pytest
import torch

from mamba_metal_scan_amd import distill_loss, linear_cross_entropy, linear_distill_loss

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (1 << 31))


def _operands(rows, dim, vocab, dtype, seed=0):
    g = _gen(rows, dim, vocab, seed)
    h = torch.randn(rows, dim, generator=g, device=DEV).to(dtype)
    w = (3.0 / math.sqrt(dim) * torch.randn(vocab, dim, generator=g, device=DEV)).to(dtype)
    return h, w, torch.randint(0, vocab, (rows,), generator=g, device=DEV)


@pytest.mark.parametrize("bad", [-math.inf, math.inf, math.nan])
@pytest.mark.parametrize("rows", [5, 40, 300])
@pytest.mark.parametrize("dtype", TYPES)
def test_ignored_rows_beside_words_of_infinity(dtype, rows, bad):
    """A row that does not count gets zeros, whatever the weight holds."""
    print(f"[case] {dtype} {rows} {bad}", flush=True)
    h, w, t = _operands(rows, 64, 300, TYPES[dtype])
    w[7, 3] = bad
    out = torch.zeros(rows, dtype=torch.bool, device=DEV)
    out[1::3] = True
    t = torch.where(out, -100, t)
    for most in (0, 1 << 30):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = linear_cross_entropy(a, b, t, reduction="none", logits_bytes=most)
        ga, gb = torch.autograd.grad(loss, [a, b], torch.ones_like(loss))
        assert (loss[out] == 0).all() and (ga[out] == 0).all()
        ids = torch.where(out[:, None], -1, torch.arange(4, device=DEV).expand(rows, 4))
        loss = linear_distill_loss(a, b, torch.zeros(rows, 4, device=DEV), ids,
                                   reduction="none", logits_bytes=most)
        ga, gb = torch.autograd.grad(loss, [a, b], torch.ones_like(loss))
        assert (loss[out] == 0).all() and (ga[out] == 0).all()


@pytest.mark.parametrize("most", [0, 1 << 30])
@pytest.mark.parametrize("dtype", TYPES)
def test_saved_tensors_in_another_layout(dtype, most):
    """Saved tensors that a hook gives back strided: the same gradients."""
    h, w, t = _operands(70, 64, 301, TYPES[dtype])
    ids = torch.arange(4, device=DEV).repeat(70, 1)
    values = torch.randn(70, 4, generator=_gen(1), device=DEV)

    def strided(x):
        if x.dim() == 2:
            return x.t().contiguous().t()
        wide = x.new_empty(2 * x.numel())
        wide[::2] = x
        return wide[::2]

    def both(pack):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        z = (h.float() @ w.float().t()).to(TYPES[dtype]).requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda x: x):
            losses = (linear_cross_entropy(a, b, t, logits_bytes=most),
                      linear_distill_loss(a, b, values, ids, logits_bytes=most),
                      distill_loss(z, values, ids))
        return [g for loss, leaves in zip(losses, ([a, b], [a, b], [z]))
                for g in torch.autograd.grad(loss, leaves)]
    for x, y in zip(both(strided), both(lambda x: x)):
        assert torch.equal(x, y)
