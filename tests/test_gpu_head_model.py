"""TinyMamba's losses from its hidden states: the same as through its logits,
gradients of every parameter (the tied head's among them), and training from
them together."""
from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

from mamba_metal_scan_amd import MambaConfig, TinyMamba, distill_loss

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _model(**kw):
    torch.manual_seed(0)
    cfg = MambaConfig(vocab_size=601, d_model=64, n_layers=2, d_ff=256, scan_impl="hip", **kw)
    return TinyMamba(cfg).to(DEV)


def _batch(seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    idx = torch.randint(0, 601, (3, 41), generator=g, device=DEV)
    x, t = idx[:, :-1].contiguous(), idx[:, 1:].clone()
    t[0, :7] = -100
    return x, t


def _grads(model, loss):
    model.zero_grad(set_to_none=True)
    loss.backward()
    return {k: p.grad.clone() for k, p in model.named_parameters()}


def _close(a, b, rel):
    scale = max(float(v.abs().max()) for v in b.values())
    for k in b:
        assert float((a[k] - b[k]).abs().max()) <= rel * max(float(b[k].abs().max()),
                                                             1e-3 * scale), k


def test_loss_matches_forward():
    """fp32 both ways: the bar of the model's other paths (1e-4)."""
    model = _model()
    x, t = _batch()
    want = model(x, t)[1]
    g_want = _grads(model, want)
    got = model.loss(x, t)
    g_got = _grads(model, got)
    assert abs(float(got) - float(want)) <= 1e-5 * float(want)
    _close(g_got, g_want, 1e-4)
    rows = model.loss(x, t, reduction="none")
    assert rows.shape == t.shape and (rows[0, :7] == 0).all()
    assert abs(float(rows.sum() / (t != -100).sum()) - float(want)) <= 1e-5 * float(want)


def test_loss_without_the_kernels():
    """scan_impl 'torch' and a hooked head take the framework's loss."""
    model = _model()
    x, t = _batch()
    want = float(model.loss(x, t))
    plain = copy.deepcopy(model)
    plain.cfg = copy.copy(model.cfg)
    plain.cfg.scan_impl = "torch"
    assert abs(float(plain.loss(x, t)) - want) <= 1e-5 * want
    seen = []
    model.head.register_forward_hook(lambda m, a, o: seen.append(o.shape))
    assert abs(float(model.loss(x, t)) - want) <= 1e-5 * want and seen


def test_distill_matches_the_logits():
    model = _model()
    x, _ = _batch()
    g = torch.Generator(device=DEV).manual_seed(3)
    values, ids = (3 * torch.randn(3, 40, 601, generator=g, device=DEV)).topk(12, dim=-1)
    ids[0, 0] = -1
    want = distill_loss(model(x)[0], values, ids, temperature=2.0)
    g_want = _grads(model, want)
    got = model.distill(x, values, ids, temperature=2.0)
    g_got = _grads(model, got)
    assert abs(float(got) - float(want)) <= 1e-5 * float(want)
    _close(g_got, g_want, 1e-4)


def test_together_under_autocast():
    """Both losses of one batch, in bf16 under autocast, summed and differentiated
    together; against the losses of the bf16 logits in fp32, whose own rounding
    (2^-9 of logits below 4) is what sets them apart."""
    model = _model()
    x, t = _batch()
    g = torch.Generator(device=DEV).manual_seed(4)
    values, ids = (3 * torch.randn(3, 40, 601, generator=g, device=DEV)).topk(8, dim=-1)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = 0.5 * model.loss(x, t) + 0.5 * model.distill(x, values, ids, temperature=2.0)
        logits = model(x)[0].float()
    g_got = _grads(model, got)
    want = 0.5 * F.cross_entropy(logits.view(-1, 601), t.view(-1)) \
        + 0.5 * distill_loss(logits, values, ids, temperature=2.0)
    assert abs(float(got) - float(want)) <= 0.03 * float(want)
    assert all(torch.isfinite(v).all() for v in g_got.values())
