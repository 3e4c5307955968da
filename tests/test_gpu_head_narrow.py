"""GPU parity of the head's losses at narrow heads (one k tile of 64) with several
tiles of 256 words x 256 rows to a block, whose rows change from tile to tile
(test_head_stream.py counts them): against 64 bits, the logits formed twice. Bounds:
head_reference.py."""
from __future__ import annotations

import math

import pytest
import torch

from head_reference import assert_head
from mamba_metal_scan_amd import linear_cross_entropy, linear_distill_loss

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _operands(rows, dim, vocab, dtype):
    """Rows whose log-sum-exps differ by up to 4, a tenth of them ignored."""
    g = torch.Generator(device=DEV).manual_seed(rows + dim + vocab)
    size = torch.linspace(0.2, 1.5, rows, device=DEV)[torch.randperm(rows, generator=g,
                                                                     device=DEV)]
    h = (size[:, None] * torch.randn(rows, dim, generator=g, device=DEV)).to(dtype)
    w = (2.0 / math.sqrt(dim) * torch.randn(vocab, dim, generator=g, device=DEV)).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    out = torch.rand(rows, generator=g, device=DEV) < 0.1
    up = torch.randn(rows, generator=g, device=DEV)
    return h, w, t, out, up


def _run(f, h, w, up, *args, **kw):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = f(h, w, *args, logits_bytes=0, **kw)
    return loss.detach(), *torch.autograd.grad(loss, [h, w], up)


# (fp32 runs other kernels, a block per tile: one size)
@pytest.mark.parametrize("dtype,rows,dim,vocab",
                         [(d, *s) for s in ((3000, 64, 32768), (700, 64, 50257),
                                            (768, 56, 131072), (2560, 8, 16384),
                                            (6000, 40, 20000), (3000, 72, 32768),
                                            (700, 128, 50257))
                          for d in ("bf16", "f16")] + [("f32", 700, 64, 50257)])
def test_rows_of_every_tile(dtype, rows, dim, vocab):
    print(f"[case] narrow {dtype} {rows}x{dim}x{vocab}", flush=True)
    h, w, t, out, up = _operands(rows, dim, vocab, TYPES[dtype])
    t = torch.where(out, -100, t)
    got = _run(linear_cross_entropy, h, w, up, t, reduction="none")
    assert (got[1][out] == 0).all()
    assert_head("xent", got, h, w, up, "none", TYPES[dtype], targets=t)
    again = _run(linear_cross_entropy, h, w, up, t, reduction="none")
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    g = torch.Generator(device=DEV).manual_seed(1)
    ids = torch.randint(0, vocab, (rows, 5), generator=g, device=DEV)
    ids[out] = -1
    values = torch.randn(rows, 5, generator=g, device=DEV)
    got = _run(linear_distill_loss, h, w, up.mean(), values, ids, temperature=2.0)
    assert (got[1][out] == 0).all()
    assert_head("distill", got, h, w, up.mean(), "mean", TYPES[dtype], words=(values, ids, 2.0))
