"""How the head's losses sit in autograd, on the CPU: the kernels' calls are replaced
by recorders, the checks of the device taken out."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from mamba_metal_scan_amd import (_native, distill_loss, head, linear_cross_entropy,
                                  linear_distill_loss)
from mamba_metal_scan_amd._native import HipScanError

ROWS, DIM, VOCAB, TOP = 6, 16, 41, 3


@pytest.fixture
def calls(monkeypatch):
    """Every kernel call's (name, arguments); forwards give zeros of the ops' shapes,
    backwards zero gradients."""
    seen = []

    def fwd(name, tops):
        def call(a, *args):
            seen.append((name, (a, *args)))
            red = args[-2] if name != "distill_fwd" else args[-1]
            n = _native._saved_size(a.shape[0], *tops)
            return torch.zeros((a.shape[0],) if red == 0 else ()), torch.zeros(n)
        return call

    def bwd(name):
        def call(grad, a, b, *args):
            seen.append((name, (grad, a, b, *args)))
            if name == "distill_bwd":
                return torch.zeros(a.shape)
            return torch.zeros(a.shape), torch.zeros(b.shape)
        return call
    for name, tops in (("linear_xent_fwd", (1,)), ("linear_distill_fwd", (TOP, TOP)),
                       ("distill_fwd", (TOP,))):
        monkeypatch.setitem(_native._IMPLS, name, fwd(name, tops))
    for name in ("linear_xent_bwd", "linear_distill_bwd", "distill_bwd"):
        monkeypatch.setitem(_native._IMPLS, name, bwd(name))
    monkeypatch.setattr(head, "_hip", lambda *a: None)
    monkeypatch.setattr(_native, "_on_one_device", lambda *a: None)
    return seen


def _losses():
    """(name, loss of the leaves, the leaves) of each of the three."""
    h, w = torch.randn(ROWS, DIM), torch.randn(VOCAB, DIM)
    t = torch.arange(ROWS)
    values, ids = torch.randn(ROWS, TOP), torch.arange(ROWS * TOP).view(ROWS, TOP)
    return [("xent", lambda a, b: linear_cross_entropy(a, b, t, logits_bytes=0), [h, w]),
            ("linear distill",
             lambda a, b: linear_distill_loss(a, b, values, ids, logits_bytes=0), [h, w]),
            ("distill", lambda a: distill_loss(a, values, ids), [torch.randn(ROWS, VOCAB)])]


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(which, grad, calls):
    """A tangent is not left out: with and without a leaf that requires grad, also
    where gradients are off."""
    _, loss, leaves = _losses()[which]
    for i in range(len(leaves)):
        for needs in (False, True):
            with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                args = [x.clone().requires_grad_(needs) for x in leaves]
                args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="jvp"):
                    loss(*args)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_alone_without_a_gradient(which, calls):
    _, loss, leaves = _losses()[which]
    assert not loss(*leaves).requires_grad
    with torch.no_grad():
        assert not loss(*(x.clone().requires_grad_() for x in leaves)).requires_grad
    assert loss(*(x.clone().requires_grad_() for x in leaves)).requires_grad
    assert len(calls) == 3


def _strided(t):
    """t's values in a layout of another kind: every second element, or transposed."""
    if t.dim() == 2:
        return t.t().contiguous().t()
    wide = t.new_empty(2 * t.numel())
    wide[::2] = t
    return wide[::2]


def _backward(loss, leaves, pack):
    args = [x.clone().requires_grad_() for x in leaves]
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = loss(*args)
    return torch.autograd.grad(out, args)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_saved_tensors_in_another_layout(which, calls):
    """What a saved-tensor hook gives back strided reaches the kernel dense."""
    _, loss, leaves = _losses()[which]
    _backward(loss, leaves, _strided)
    name, args = calls[-1]
    tensors = [a for a in args if isinstance(a, torch.Tensor)]
    assert name.endswith("_bwd") and len(tensors) == (4 if which == 2 else 5)
    for t in tensors:
        assert t.is_contiguous() and t.data_ptr() % 16 == 0
    want = [x for x in leaves]
    for got, x in zip(tensors[1:], want):
        assert torch.equal(got, x)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("what", ["half", "int32", "short"])
def test_saved_tensors_that_changed_are_refused(which, what, calls):
    """Of another type or size they would be read past their end."""
    def pack(t):
        if what == "half":
            return t.bfloat16() if t.dtype == torch.float32 and t.dim() == 1 else t
        if what == "int32":
            return t.int() if t.dtype == torch.int64 else t
        return t[:-1] if t.dim() == 1 else t[:, :-1] if t.dtype == torch.int64 else t
    _, loss, leaves = _losses()[which]
    with pytest.raises(HipScanError):
        _backward(loss, leaves, pack)
    assert not any(name.endswith("_bwd") for name, _ in calls)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("dynamic", [None, True])
def test_traced_in_one_graph(which, dynamic, monkeypatch):
    """torch.compile takes each loss whole (fullgraph), as the package's other ops."""
    monkeypatch.setattr(head, "_hip", lambda *a: None)
    graphs = []

    def backend(gm, example):
        graphs.append(gm)
        return lambda *a: [torch.zeros(())]
    _, loss, leaves = _losses()[which]
    torch._dynamo.reset()
    with torch.no_grad():
        torch.compile(loss, backend=backend, fullgraph=True, dynamic=dynamic)(*leaves)
    op = ("linear_xent_fwd", "linear_distill_fwd", "distill_fwd")[which]
    assert len(graphs) == 1 and f"mamba_hip.{op}" in graphs[0].code
    torch.compile(loss, backend=backend, fullgraph=True, dynamic=dynamic)(
        *(x.requires_grad_() for x in leaves))
    assert len(graphs) == 2
    torch._dynamo.reset()


@pytest.mark.parametrize("layout", ["transposed", "sliced"])
def test_a_vocabulary_of_one_word(layout, calls):
    """Logits (rows, 1) whose last stride is not 1: contiguous by torch's account."""
    z = torch.randn(1, ROWS).t() if layout == "transposed" else torch.randn(1, 3)[:, ::3]
    rows = z.shape[0]
    values, ids = torch.randn(rows, TOP), torch.zeros(rows, TOP, dtype=torch.int64)
    distill_loss(z, values, ids)
    assert calls[-1][1][0].stride() == (1, 1)
