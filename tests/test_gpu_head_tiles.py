"""GPU parity of the head's losses at the edges of the 16-bit products' tiles (256 words
x 256 rows) and of the fp32 ones' (128 x 128), over one round of the CUs and more, and the
gradients' errors in the norm. Bounds: head_reference.py."""
from __future__ import annotations

import math

import pytest
import torch

from head_reference import Reference, assert_head
from mamba_metal_scan_amd import _native, linear_cross_entropy, linear_distill_loss

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (1 << 31))


def _operands(rows, dim, vocab, dtype, spread=2.0):
    g = _gen(rows, dim, vocab)
    h = torch.randn(rows, dim, generator=g, device=DEV).to(dtype)
    w = (spread / math.sqrt(dim) * torch.randn(vocab, dim, generator=g, device=DEV)).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    return h, w, torch.where(torch.rand(rows, generator=g, device=DEV) < 0.1, -100, t)


def _words(rows, vocab, k):
    g = _gen(rows, vocab, k, 1)
    ids = torch.rand(rows, vocab, generator=g, device=DEV).topk(k, dim=1).indices
    values = 2.0 * torch.randn(rows, k, generator=g, device=DEV)
    ids[::7] = -1
    return values, ids


def _run(f, h, w, up, *args, **kw):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = f(h, w, *args, **kw)
    return loss.detach(), *torch.autograd.grad(loss, [h, w], up)


@pytest.mark.parametrize("most", [0, 1 << 30])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(255, 128, 257), (256, 64, 256), (257, 192, 255),
                                            (128, 72, 129), (511, 64, 513), (512, 136, 1023),
                                            (513, 64, 1281), (769, 128, 769)])
def test_edges_of_tiles(rows, dim, vocab, dtype, most):
    print(f"[case] tiles {dtype} {rows}x{dim}x{vocab} {most}", flush=True)
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    up = torch.randn(rows, generator=_gen(rows), device=DEV)
    got = _run(linear_cross_entropy, h, w, up, t, reduction="none", logits_bytes=most)
    assert_head("xent", got, h, w, up, "none", TYPES[dtype], targets=t)
    words = _words(rows, vocab, 6)
    up = torch.ones((), device=DEV)
    got = _run(linear_distill_loss, h, w, up, *words, temperature=1.5, logits_bytes=most)
    assert_head("distill", got, h, w, up, "mean", TYPES[dtype], words=(*words, 1.5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(700, 128, 50257), (1300, 192, 16390),
                                            (300, 384, 65537)])
def test_more_tiles_than_compute_units(rows, dim, vocab, dtype):
    """Row tiles that are no power of two (3, 6 and 2), a last round of a few tiles."""
    print(f"[case] rounds {dtype} {rows}x{dim}x{vocab}", flush=True)
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    up = torch.randn(rows, generator=_gen(rows), device=DEV)
    got = _run(linear_cross_entropy, h, w, up, t, reduction="none", logits_bytes=0)
    assert_head("xent", got, h, w, up, "none", TYPES[dtype], targets=t)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("words", [0, 64])
@pytest.mark.parametrize("rows,dim,vocab", [(1001, 384, 50257), (1024, 640, 32768)])
def test_errors_in_the_norm(rows, dim, vocab, words, dtype):
    """What the elementwise bounds, which add every term's error by its size, leave
    open. Each rounding to 16 bits, of the logits' gradient and of the result, is off by
    at most u = half a unit of the power of two below the value, u / sqrt(3) on the mean
    of squares where errors are spread evenly and independent (a common factor kept
    out of the rounding is what makes them so): of dh
      sum (u^2 / 3) (dz^2 W^2) + (u^2 / 3) dh^2,
    a bound on the expectation, since values lie above their power of two. Over 4e5
    and more elements the sum of squares is within 1% of it; fp32's part (2^-17 of p) is
    another 1% of u in bf16, a tenth in fp16: 12% in all."""
    dt = TYPES[dtype]
    h, w, t = _operands(rows, dim, vocab, dt)
    up = torch.full((), 0.7, device=DEV)   # no power of two
    hd, wd = h.double(), w.double()
    z = hd @ wd.t()
    if words:
        kind = dict(words=(*_words(rows, vocab, words), 2.0))
        got = _run(linear_distill_loss, h, w, up, *kind["words"][:2], temperature=2.0)
    else:
        kind = dict(targets=t)
        got = _run(linear_cross_entropy, h, w, up, t)
    ref = Reference(z, torch.zeros_like(z), **kind)
    dz = ref.dz * (0.7 * ref.reduced("mean")[2])
    u = torch.finfo(dt).eps / 2
    for name, g, a, b in (("dh", got[1], dz, wd), ("dW", got[2], dz.t().contiguous(), hd)):
        want = a @ b
        off = (g.double() - want).norm()
        sizes = u * u * ((a.square() @ b.square()).sum() + want.square().sum())
        if dt == torch.float16:   # (below its normal numbers a result's half step is 2^-25)
            sizes = sizes + 2.0 ** -50 * want.numel()
        most = (sizes / 3).sqrt()
        print(f"{name} {float(off / want.norm()):.3g} of {float(most / want.norm()):.3g}")
        assert off <= 1.12 * most, (name, float(off), float(most))


def test_leading_dimensions_of_distillation():
    h, w, _ = _operands(60, 64, 200, torch.float32)
    values, ids = _words(60, 200, 8)
    want = linear_distill_loss(h, w, values, ids, reduction="none")
    got = linear_distill_loss(h.view(3, 20, 64), w, values.view(3, 20, 8),
                              ids.view(3, 20, 8).int(), reduction="none")
    assert got.shape == (3, 20) and torch.equal(got.view(-1), want)


def test_autocast_takes_the_losses_from_hidden_states(monkeypatch):
    """Under autocast the model's losses run on the head's kernels, in its type."""
    from mamba_metal_scan_amd import MambaConfig, TinyMamba
    torch.manual_seed(0)
    model = TinyMamba(MambaConfig(vocab_size=601, d_model=64, n_layers=1, d_ff=256,
                                  scan_impl="hip")).to(DEV)
    x = torch.randint(0, 601, (3, 40), generator=_gen(3), device=DEV)
    ids = torch.randint(0, 601, (3, 40, 5), generator=_gen(4), device=DEV)
    values = torch.randn(3, 40, 5, generator=_gen(5), device=DEV)
    seen = []
    for name in ("linear_xent_fwd", "linear_distill_fwd", "linear_xent_bwd",
                 "linear_distill_bwd"):
        def call(*args, _f=_native._IMPLS[name], _name=name, **kw):
            seen.append((_name, args[1].dtype))
            return _f(*args, **kw)
        monkeypatch.setitem(_native._IMPLS, name, call)
    for dt in (torch.bfloat16, None):   # (the scan takes no fp16)
        seen.clear()
        with torch.autocast("cuda", dtype=dt, enabled=dt is not None):
            loss = model.loss(x, x) + model.distill(x, values, ids)
        loss.backward()
        assert sorted(n for n, _ in seen) == ["linear_distill_bwd", "linear_distill_fwd",
                                              "linear_xent_bwd", "linear_xent_fwd"]
        assert all(d == (dt or torch.float32) for _, d in seen)
        assert loss.dtype == torch.float32
        assert all(torch.isfinite(p.grad).all() for p in model.parameters())
