"""Losses of TinyMamba's head from its hidden states, on the HIP kernels.

The reference forms the head's logits and takes their cross entropy
(mamba_metal/model.py:294-297): at the 80M model's batch (8192 rows x 32768
words) 1.07 GB of fp32 logits and as much again for their gradient.
``linear_cross_entropy`` computes the same loss and both gradients from the
hidden states and the head's weight, the logits formed tile by tile on the
matrix cores: the forward reduces each tile to its rows' maxima and sums of
exponentials, the backward forms the tiles again, a piece of the vocabulary at a
time, and multiplies their gradient with the weight and the hidden states.

What a training call holds. From forward to backward, by default, up to 1 GiB
(``logits_bytes``) of fp32 logits, where their total fits that and keeping them is the
faster: always in fp32, so all of the batch above's 2^30 bytes, and up to 256 rows or from 2048
columns in 16 bits. ``logits_bytes=0`` holds none, for a fourth product (at that batch in
fp32 7330 us where 5980). During the backward up to 256 MB of the logits' gradient. Without
a backward nothing is kept.

``distill_loss`` is the distillation of given logits from a teacher's top words,
``linear_distill_loss`` the same from the hidden states.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.forward_ad import unpack_dual

from . import _native
from ._native import REDUCE, HipScanError, dispatch


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """The 2-D t, or a copy of it whose rows the kernels read in place (zeros
    in the columns that fill up its rows). While tracing of the right layout: the ops
    see to the alignment, which is known only then."""
    if (_native.head_layout if torch.compiler.is_compiling() else _native.head_rows)(t):
        return t
    pad = -t.shape[1] % (16 // t.element_size())
    return F.pad(t, (0, pad)) if pad else t.clone(memory_format=torch.contiguous_format)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The 2-D t, or a copy of it with contiguous rows that do not overlap."""
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        # (contiguous() would leave the strides of a single column as they are)
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _cut(g: torch.Tensor, dim: int) -> torch.Tensor:
    """A gradient without the columns that _rows16 added."""
    return g if g.shape[1] == dim else g[:, :dim].contiguous()


LOGITS_BYTES = 1 << 30   # of fp32 logits that a forward may keep, unless told otherwise


def _keeps(hidden: torch.Tensor, weight: torch.Tensor, most: int) -> bool:
    return _native.keeps_logits(hidden.shape[0], weight.shape[0], hidden.shape[1], hidden.dtype,
                                most)


def _layout(ts) -> list:
    return [(t.dtype, t.device, t.shape, t.stride()) for t in ts]


def _save(ctx, ts) -> None:
    ctx.save_for_backward(*ts)
    ctx.layout = None if torch.compiler.is_compiling() else _layout(ts)


def _restored(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _saved(ctx, rows, check) -> tuple:
    """The saved tensors as the kernels read them (the last one 16-byte aligned). A
    saved-tensor hook may give them back in another layout, or changed: then matrices of
    floats go through rows, the others are made dense, and check(*them) refuses what the
    kernels would read past its end."""
    ts = ctx.saved_tensors
    if ctx.layout is None or torch.compiler.is_compiling() \
            or (_layout(ts) == ctx.layout and ts[-1].data_ptr() % 16 == 0):
        return ts
    ts = tuple((rows if t.dim() == 2 and t.is_floating_point() else _restored)(t) for t in ts)
    check(*ts)
    return ts


def _once() -> None:
    """The gradients have none of their own: refuses a backward that is to be
    differentiated (create_graph) rather than leave their part out."""
    if torch.is_grad_enabled() and not torch.compiler.is_compiling():
        raise HipScanError("the head's losses are once differentiable (create_graph is not "
                           "supported); take the loss of the logits instead")


def _grads(ctx, dhidden: torch.Tensor, dweight: torch.Tensor):
    return (_cut(dhidden, ctx.dim) if ctx.needs_input_grad[0] else None,
            _cut(dweight, ctx.dim) if ctx.needs_input_grad[1] else None)


class LinearCrossEntropyHIP(torch.autograd.Function):
    """Cross entropy of hidden (R, D) weight (V, D)^T against targets (R)
    int64; rows with target == ignore_index excluded."""

    @staticmethod
    def loss(hidden, weight, targets, ignore_index, reduction, most, backward=False):
        """(loss, what the backward needs)."""
        hidden, weight = _rows16(hidden), _rows16(weight)
        targets = targets.contiguous()
        if not torch.compiler.is_compiling():   # (the registered op checks itself)
            _native._check_linear_xent("linear_cross_entropy", hidden, weight, targets, reduction)
        loss, saved = dispatch("linear_xent_fwd")(hidden, weight, targets, ignore_index, reduction,
                                                  backward and _keeps(hidden, weight, most))
        return loss, (hidden, weight, targets, saved)

    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction, most):
        ctx.dim = hidden.shape[1]
        ctx.reduction = reduction
        loss, saved = LinearCrossEntropyHIP.loss(hidden, weight, targets, ignore_index, reduction,
                                                 most, any(ctx.needs_input_grad))
        _save(ctx, saved)
        return loss

    @staticmethod
    def backward(ctx, g):
        _once()
        g = g.contiguous()
        rest = (ctx.reduction, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        ts = _saved(ctx, _rows16, lambda *ts: _native._check_linear_xent_bwd(g, *ts, *rest))
        return (*_grads(ctx, *dispatch("linear_xent_bwd")(g, *ts, *rest)), None, None, None, None)


class LinearDistillHIP(torch.autograd.Function):
    """Distillation of hidden (R, D) weight (V, D)^T from the teacher's words
    ids (R, K) and their logits."""

    @staticmethod
    def loss(hidden, weight, teacher_logits, ids, temperature, reduction, most, backward=False):
        """(loss, what the backward needs)."""
        hidden, weight = _rows16(hidden), _rows16(weight)
        if not torch.compiler.is_compiling():
            _native._check_linear_distill("linear_distill_loss", hidden, weight, teacher_logits,
                                          ids, temperature, reduction)
        loss, saved = dispatch("linear_distill_fwd")(hidden, weight, teacher_logits, ids,
                                                     temperature, reduction,
                                                     backward and _keeps(hidden, weight, most))
        return loss, (hidden, weight, ids, saved)

    @staticmethod
    def forward(ctx, hidden, weight, teacher_logits, ids, temperature, reduction, most):
        ctx.dim = hidden.shape[1]
        ctx.temperature, ctx.reduction = temperature, reduction
        loss, saved = LinearDistillHIP.loss(hidden, weight, teacher_logits, ids, temperature,
                                            reduction, most, any(ctx.needs_input_grad))
        _save(ctx, saved)
        return loss

    @staticmethod
    def backward(ctx, g):
        _once()
        g = g.contiguous()
        rest = (ctx.temperature, ctx.reduction, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        ts = _saved(ctx, _rows16, lambda *ts: _native._check_linear_distill_bwd(g, *ts, *rest))
        return (*_grads(ctx, *dispatch("linear_distill_bwd")(g, *ts, *rest)),
                None, None, None, None, None)


class DistillHIP(torch.autograd.Function):
    """Distillation of logits (R, V) from the teacher's words ids (R, K) and
    their logits."""

    @staticmethod
    def loss(logits, teacher_logits, ids, temperature, reduction):
        """(loss, what the backward needs)."""
        logits = _rows(logits)
        if not torch.compiler.is_compiling():
            _native._check_distill("distill_loss", logits, teacher_logits, ids, temperature,
                                   reduction)
        loss, saved = dispatch("distill_fwd")(logits, teacher_logits, ids, temperature, reduction)
        return loss, (logits, ids, saved)

    @staticmethod
    def forward(ctx, logits, teacher_logits, ids, temperature, reduction):
        ctx.temperature, ctx.reduction = temperature, reduction
        loss, saved = DistillHIP.loss(logits, teacher_logits, ids, temperature, reduction)
        _save(ctx, saved)
        return loss

    @staticmethod
    def backward(ctx, g):
        _once()
        g = g.contiguous()
        rest = (ctx.temperature, ctx.reduction)
        ts = _saved(ctx, _rows, lambda *ts: _native._check_distill_bwd(g, *ts, *rest))
        return dispatch("distill_bwd")(g, *ts, *rest), None, None, None, None


def _recorded(ts) -> bool:
    """Whether autograd records what becomes of ts: one requires grad, or has a tangent."""
    grad = torch.is_grad_enabled()
    for t in ts:
        if (grad and t.requires_grad) or unpack_dual(t).tangent is not None:
            return True
    return False


def _apply(cls, leaves: int, *args):
    """cls.apply, or without autograd to record (scoring, serving) its forward
    alone. (Leaves with a tangent go to apply, which refuses forward-mode
    derivatives: its forward alone would leave them out.)"""
    if torch.compiler.is_compiling() or _recorded(args[:leaves]):
        return cls.apply(*args)
    return cls.loss(*args)[0]


def _reduction(what: str, reduction: str) -> int:
    if reduction not in REDUCE:
        raise ValueError(f"{what}: reduction must be 'mean', 'sum' or 'none'; got {reduction!r}")
    return REDUCE[reduction]


def _bytes(what: str, n: int) -> int:
    if not isinstance(n, int) or n < 0:
        raise ValueError(f"{what}: logits_bytes must be an integer of at least 0; got {n!r}")
    return n


def _hip(what: str, *ts: torch.Tensor) -> None:
    if torch.version.hip is None or not all(t.is_cuda for t in ts):
        raise RuntimeError(f"{what} needs its tensors on the ROCm device; got "
                           + ", ".join(str(t.device) for t in ts))


def _head(what: str, hidden: torch.Tensor, weight: torch.Tensor):
    """hidden as (rows, dim), and weight; both in autocast's type where that is
    enabled, as the head's linear layer takes them."""
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: hidden must be (..., dim) and weight (vocab, dim); got "
                         f"{tuple(hidden.shape)}, {tuple(weight.shape)}")
    if 0 in weight.shape:
        raise ValueError(f"{what}: weight must not be empty; got {tuple(weight.shape)}")
    if torch.is_autocast_enabled():
        t = torch.get_autocast_dtype("cuda")
        hidden, weight = hidden.to(t), weight.to(t)
    if hidden.dtype != weight.dtype or hidden.dtype not in _native.HEAD_DTYPES:
        raise RuntimeError(f"{what}: hidden and weight must both be float32, bfloat16 or "
                           f"float16; got {hidden.dtype}, {weight.dtype}")
    return hidden.reshape(-1, hidden.shape[-1]), weight


def _teacher(what: str, lead: torch.Size, teacher_logits: torch.Tensor,
             teacher_ids: torch.Tensor, temperature: float):
    """The teacher's logits (rows, k) fp32 and words (rows, k) int64, contiguous."""
    if (teacher_ids.dim() < 1 or teacher_ids.shape != teacher_logits.shape
            or teacher_ids.shape[:-1] != lead):
        raise ValueError(f"{what}: teacher_logits and teacher_ids must be {tuple(lead)} + (k,); "
                         f"got {tuple(teacher_logits.shape)}, {tuple(teacher_ids.shape)}")
    k = teacher_ids.shape[-1]
    if not 1 <= k <= _native.MAX_TOP:
        raise ValueError(f"{what}: the teacher's words per row must be in "
                         f"[1, {_native.MAX_TOP}]; got {k}")
    if teacher_ids.is_floating_point() or teacher_ids.is_complex() \
            or teacher_ids.dtype == torch.bool or not teacher_logits.is_floating_point():
        raise RuntimeError(f"{what}: teacher_ids must be integers and teacher_logits floating "
                           f"point; got {teacher_ids.dtype}, {teacher_logits.dtype}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"{what}: temperature must be positive and finite; got {temperature}")
    return (teacher_logits.detach().to(torch.float32).reshape(-1, k).contiguous(),
            teacher_ids.to(torch.int64).reshape(-1, k).contiguous())


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                         ignore_index: int = -100, reduction: str = "mean",
                         logits_bytes: int = LOGITS_BYTES) -> torch.Tensor:
    """``F.cross_entropy(hidden @ weight.T, targets, ignore_index=ignore_index,
    reduction=reduction)`` from the operands: hidden (..., D) and weight (V, D)
    in float32, bfloat16 or float16 on one ROCm device, targets (...) integers.

    The loss is float32: a scalar, or with reduction "none" one per row, of
    targets' shape (0 where ignored). Rows that are ignored add nothing to the
    gradients, whatever they hold. A target outside [0, V) that is not
    ignore_index makes its row's loss NaN. Fp32 logits (rows x V x 4 bytes) that take
    no more than logits_bytes, 1 GiB unless given, may be kept whole from forward to
    backward, where that is the faster; 0 keeps none. Under autocast hidden and weight are
    taken in its type. Logits are meant to lie within 2^20: a probability is off by 2^-24
    of their size. The gradients are once differentiable."""
    what = "linear_cross_entropy"
    _hip(what, hidden, weight, targets)
    red = _reduction(what, reduction)
    if targets.shape != hidden.shape[:-1] or targets.is_floating_point() \
            or targets.is_complex() or targets.dtype == torch.bool:
        raise ValueError(f"{what}: targets must be integers of shape {tuple(hidden.shape[:-1])}; "
                         f"got {targets.dtype} {tuple(targets.shape)}")
    h, w = _head(what, hidden, weight)
    loss = _apply(LinearCrossEntropyHIP, 2, h, w, targets.to(torch.int64).reshape(-1),
                  int(ignore_index), red, _bytes(what, logits_bytes))
    return loss if red else loss.view(targets.shape)


def linear_distill_loss(hidden: torch.Tensor, weight: torch.Tensor,
                        teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                        temperature: float = 1.0, reduction: str = "mean",
                        logits_bytes: int = LOGITS_BYTES) -> torch.Tensor:
    """``distill_loss(hidden @ weight.T, ...)`` from the operands: hidden (..., D),
    weight (V, D) and logits_bytes as linear_cross_entropy takes them,
    teacher_logits and teacher_ids (..., K)."""
    what = "linear_distill_loss"
    _hip(what, hidden, weight, teacher_logits, teacher_ids)
    red = _reduction(what, reduction)
    temperature = float(temperature)
    lead = hidden.shape[:-1]
    t, ids = _teacher(what, lead, teacher_logits, teacher_ids, temperature)
    h, w = _head(what, hidden, weight)
    loss = _apply(LinearDistillHIP, 2, h, w, t, ids, temperature, red, _bytes(what, logits_bytes))
    return loss if red else loss.view(lead)


def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                 temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """Distillation of the student's logits (..., V) (float32, bfloat16 or
    float16) from a teacher's top words: teacher_ids (..., K) and their
    teacher_logits, K up to 1024, an id below 0 being padding.

    With q = softmax(teacher_logits / temperature) over a row's kept words and
    p = softmax(logits / temperature) over the vocabulary, a row's loss is
    temperature^2 sum_k q_k (log q_k - log p_k), terms with q_k = 0 being 0. A
    row of logits that are all alike, be it the type's lowest value (a mask that leaves
    nothing), is the uniform distribution; one of -inf alone is NaN. A
    row that keeps no word, or whose kept logits are all -inf, has loss 0 and no
    gradient, and the mean leaves it out (NaN where it leaves out all); an id at
    or past V makes its row's loss NaN; a word named twice has both weights. The
    teacher gets no gradient; the student's is once differentiable. The loss is
    float32: a scalar, or with reduction "none" of the rows' shape."""
    what = "distill_loss"
    _hip(what, logits, teacher_logits, teacher_ids)
    red = _reduction(what, reduction)
    temperature = float(temperature)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be (..., vocab); got {tuple(logits.shape)}")
    if logits.dtype not in _native.HEAD_DTYPES:
        raise RuntimeError(f"{what}: logits must be float32, bfloat16 or float16; got "
                           f"{logits.dtype}")
    lead = logits.shape[:-1]
    t, ids = _teacher(what, lead, teacher_logits, teacher_ids, temperature)
    loss = _apply(DistillHIP, 1, logits.reshape(-1, logits.shape[-1]), t, ids, temperature, red)
    return loss if red else loss.view(lead)
