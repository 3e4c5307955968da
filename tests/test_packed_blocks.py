"""Packed sequences through a model whose blocks are not plain: mix_packed() takes the place of a
call of the block and reads the conv's weights, so that what a hook, a subclass, a wrapper or a
method set on the instance would do is refused and not left out."""
from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from torch.nn.utils import parametrize

from helpers import assert_close
from mamba_metal_scan_amd.model import MambaBlock, MambaConfig, TinyMamba

VOCAB = 61


def _model():
    torch.manual_seed(3)
    return TinyMamba(MambaConfig(vocab_size=VOCAB, d_model=64, n_layers=2, d_ff=128,
                                 scan_impl="hip"))


class Wrapper(nn.Module):
    def __init__(self, block):
        super().__init__()
        self.block = block

    def forward(self, x, cache=None):
        return 2 * self.block(x, cache)


class Doubled(MambaBlock):
    def mix(self, h, cache=None):
        return 2 * super().mix(h, cache)


def _hook(m):
    m.blocks[1].register_forward_hook(lambda mod, args, out: 2 * out)


def _pre_hook(m):
    m.blocks[1].register_forward_pre_hook(lambda mod, args: (2 * args[0], *args[1:]))


def _backward_hook(m):
    m.blocks[1].register_full_backward_hook(lambda mod, gi, go: None)


def _subclass(m):
    m.blocks[1].__class__ = Doubled


def _wrapper(m):
    m.blocks[1] = Wrapper(m.blocks[1])


def _forward(m):
    m.blocks[1].forward = lambda x, cache=None: 2 * x


def _mix(m):
    m.blocks[1].mix = lambda h, cache=None: 2 * h


def _scan(m):
    m.blocks[1]._scan = lambda x, return_state=False: x


def _call(m):
    m.blocks[1].__class__ = type("Called", (MambaBlock,),
                                 {"__call__": lambda self, x, cache=None: 2 * x})


def _conv_subclass(m):
    m.blocks[1].conv.__class__ = type("Scaled", (nn.Conv1d,), {"forward": lambda self, x: 2 * x})


def _conv_hook(m):
    m.blocks[1].conv.register_forward_hook(lambda mod, args, out: 2 * out)


def _conv_forward(m):
    m.blocks[1].conv.forward = lambda x: 2 * x


CHANGES = [_hook, _pre_hook, _backward_hook, _subclass, _wrapper, _forward, _mix, _scan,
           _call, _conv_subclass, _conv_hook, _conv_forward]


def _refused(m, dev):
    idx = torch.arange(9, device=dev)
    cu = torch.tensor([0, 4, 9], device=dev)
    for call in (lambda: m.prefill(idx, cu, {}), lambda: m.loss(idx, idx, cu_seqlens=cu),
                 lambda: m.generate(idx, cu, 2)):
        with pytest.raises(RuntimeError, match="block 1 .* without hooks or methods"):
            call()


@pytest.mark.parametrize("change", CHANGES)
def test_what_would_be_left_out_is_refused(change):
    m = _model()
    change(m)
    _refused(m, "cpu")


def test_global_hooks_are_refused():
    m = _model()
    handle = nn.modules.module.register_module_forward_hook(lambda mod, args, out: None)
    try:
        with pytest.raises(RuntimeError, match="block 0 .* without hooks or methods"):
            m.prefill(torch.arange(3), torch.tensor([0, 3]), {})
    finally:
        handle.remove()


@pytest.mark.gpu
@pytest.mark.parametrize("change", CHANGES)
def test_what_would_be_left_out_is_refused_on_the_gpu(change):
    m = _model().cuda()
    change(m)
    _refused(m, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["norm", "in_proj", "dt_proj", "B_proj", "C_proj", "out_proj"])
def test_modules_that_are_called_keep_their_hooks(name):
    """Those of a block's modules but the conv run: as of each document alone, through the
    blocks' path by modules (a hook of the norm, and a cache, keep the model from the others)."""
    m = _model().cuda()
    calls = []

    def hook(mod, args, out):
        calls.append(1)
        return 2 * out

    idx = torch.arange(9, device="cuda")
    with torch.no_grad():
        plain = m.prefill(idx, torch.tensor([0, 4, 9], device="cuda"), {})
        getattr(m.blocks[1], name).register_forward_hook(hook)
        got = m.prefill(idx, torch.tensor([0, 4, 9], device="cuda"), {})
        assert calls == [1]
        want = torch.stack([m(p[None], cache={})[0][0, -1] for p in (idx[:4], idx[4:])])
        assert calls == [1, 1, 1]
    assert_close("logits", got, want, 2e-5)
    assert not torch.allclose(got, plain)


class Twice(nn.Module):
    def forward(self, w):
        return 2 * w


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["conv.weight", "A", "D_skip", "in_proj.weight", "subclass"])
def test_what_leaves_the_methods_alone_is_taken(where):
    """Parametrized weights (a subclass of the module's class) are read as they are, and so is a
    subclass that overrides none of the methods: as of each document alone."""
    m = _model().cuda()
    block = m.blocks[1]
    idx = torch.arange(9, device="cuda")
    cu = torch.tensor([0, 4, 9], device="cuda")
    with torch.no_grad():
        plain = m.prefill(idx, cu, {})
    if where == "subclass":
        block.__class__ = type("Named", (MambaBlock,), {"extra": lambda self: 1})
    else:
        owner = block if "." not in where else getattr(block, where.split(".")[0])
        parametrize.register_parametrization(owner, where.split(".")[-1], Twice(), unsafe=True)
    with torch.no_grad():
        got = m.prefill(idx, cu, {})
        want = torch.stack([m(p[None], cache={})[0][0, -1] for p in (idx[:4], idx[4:])])
    assert_close("logits", got, want, 2e-5)
    assert torch.allclose(got, plain) == (where == "subclass")


@pytest.mark.gpu
def test_the_loss_of_packed_documents_is_traced():
    m = _model().cuda()
    idx = torch.arange(9, device="cuda")
    cu = torch.tensor([0, 4, 9], device="cuda")
    want = m.loss(idx, idx, cu_seqlens=cu)
    got = torch.compile(lambda i, c: m.loss(i, i, cu_seqlens=c), backend="aot_eager",
                        fullgraph=True)(idx, cu)
    assert_close("loss", got, want, 1e-6)
