"""GPU parity of the head's losses from hidden states with 64 bits: sizes at the
tiles' edges (256 words x 128 rows, 64 deep; 128 x 128 in fp32; 64 words x 16 or
32 rows for few rows), every type, reduction and direction, rows that do not
count, strides and alignments. Bounds: head_reference.py."""
from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from head_reference import UNIT, assert_head, assert_within, sum_error
from mamba_metal_scan_amd import _native, linear_cross_entropy, linear_distill_loss
from mamba_metal_scan_amd._native import HipScanError

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = {"f32": F32, "bf16": BF16, "f16": F16}


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (1 << 31))


def _operands(rows, dim, vocab, dtype, spread=3.0, seed=0):
    """h, w with logits of standard deviation `spread`, targets with a tenth
    ignored (the first kept)."""
    g = _gen(rows, dim, vocab, seed)
    h = torch.randn(rows, dim, generator=g, device=DEV).to(dtype)
    w = (spread / math.sqrt(dim) * torch.randn(vocab, dim, generator=g, device=DEV)).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    t = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.1, -100, t)
    if rows:
        t[0] = vocab - 1
    return h, w, t


def _words(rows, vocab, k, seed=0):
    """A teacher's words: distinct where the vocabulary allows, a third of the
    rows with padding, among them empty rows."""
    g = _gen(rows, vocab, k, seed, 1)
    ids = torch.rand(rows, max(vocab, k), generator=g, device=DEV).argsort(1)[:, :k] % vocab
    values = 2.0 * torch.randn(rows, k, generator=g, device=DEV)
    keep = torch.rand(rows, k, generator=g, device=DEV) < 0.6
    some = torch.rand(rows, 1, generator=g, device=DEV) < 0.33
    ids = torch.where(some & ~keep, -1, ids)
    if rows > 2:
        ids[1] = -1                      # nothing kept
        values[2] = -math.inf            # kept, but impossible
        if k > 1:
            ids[0, 1] = ids[0, 0]        # a word named twice
            values[0, -1] = -math.inf    # one impossible word
    return values, ids


def _upstream(rows, reduction, seed=0):
    g = _gen(rows, seed, 2)
    return torch.randn((rows,) if reduction == "none" else (), generator=g, device=DEV)


def _run(f, h, w, up, *args, **kw):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = f(h, w, *args, **kw)
    return loss.detach(), *torch.autograd.grad(loss, [h, w], up)


SIZES = [(1, 8, 1), (1, 64, 7), (3, 64, 257), (16, 640, 1000), (17, 128, 65), (32, 72, 256),
         (33, 64, 255), (127, 192, 300), (129, 64, 513), (300, 1024, 1001), (515, 56, 5003),
         (13, 1160, 1030), (24, 2056, 131)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", SIZES)
def test_cross_entropy(rows, dim, vocab, dtype):
    print(f"[case] linear xent {dtype} {rows}x{dim}x{vocab}", flush=True)
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    for reduction in ("mean", "sum", "none"):
        up = _upstream(rows, reduction)
        got = _run(linear_cross_entropy, h, w, up, t, reduction=reduction)
        assert_head(f"{reduction}", got, h, w, up, reduction, TYPES[dtype], targets=t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab,k,temperature",
                         [(1, 64, 7, 1, 1.0), (5, 64, 300, 5, 2.0), (33, 128, 1000, 64, 4.0),
                          (130, 192, 515, 20, 1.5), (300, 64, 3001, 128, 0.5)])
def test_distillation(rows, dim, vocab, k, temperature, dtype):
    print(f"[case] linear distill {dtype} {rows}x{dim}x{vocab} k {k}", flush=True)
    h, w, _ = _operands(rows, dim, vocab, TYPES[dtype])
    values, ids = _words(rows, vocab, k)
    for reduction in ("mean", "sum", "none"):
        up = _upstream(rows, reduction)
        got = _run(linear_distill_loss, h, w, up, values, ids, temperature=temperature,
                   reduction=reduction)
        assert_head(f"{reduction}", got, h, w, up, reduction, TYPES[dtype],
                    words=(values, ids, temperature))


def _keep(monkeypatch, keep):
    """The forward keeps its logits, or the backward forms them again."""
    monkeypatch.setattr(_native, "keeps_logits", lambda *a: keep)


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(1, 64, 1), (5, 64, 130), (17, 64, 66), (33, 64, 257),
                                            (64, 72, 1003), (65, 64, 515), (130, 64, 258),
                                            (300, 200, 1030)])
def test_logits_kept_or_formed_again(rows, dim, vocab, dtype, keep, monkeypatch):
    print(f"[case] keep {keep} {dtype} {rows}x{dim}x{vocab}", flush=True)
    _keep(monkeypatch, keep)
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    up = _upstream(rows, "none")
    got = _run(linear_cross_entropy, h, w, up, t, reduction="none")
    assert_head("xent", got, h, w, up, "none", TYPES[dtype], targets=t)
    values, ids = _words(rows, vocab, 3)
    up = _upstream(rows, "mean")
    got = _run(linear_distill_loss, h, w, up, values, ids, temperature=2.0)
    assert_head("distill", got, h, w, up, "mean", TYPES[dtype], words=(values, ids, 2.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bytes_of_logits_kept(dtype):
    """What a loss holds until its backward: the logits, or none of them."""
    h, w, t = _operands(200, 64, 40000, TYPES[dtype])
    up = torch.ones((), device=DEV)
    a, b = h.requires_grad_(), w.requires_grad_()
    held, grads = [], []
    for most in (0, 200 * 40000 * 4 - 1, 200 * 40000 * 4):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = linear_cross_entropy(a, b, t, logits_bytes=most)
        held.append(torch.cuda.memory_allocated() - before)
        grads.append(torch.autograd.grad(loss, [a, b], up))
        del loss
        assert_head(f"{most}", (linear_cross_entropy(h.detach(), w.detach(), t), *grads[-1]),
                    h.detach(), w.detach(), up, "mean", TYPES[dtype], targets=t)
    assert held[0] < 1 << 20 and held[1] < 1 << 20 and held[2] >= 200 * 40000 * 4
    for x, y in zip(grads[0], grads[1]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES)
def test_kept_logits_of_a_backward_twice(dtype, monkeypatch):
    """The backward leaves what the forward kept as it was."""
    _keep(monkeypatch, True)
    h, w, t = _operands(70, 64, 300, TYPES[dtype])
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(a, b, t)
    first = torch.autograd.grad(loss, [a, b], retain_graph=True)
    for x, y in zip(first, torch.autograd.grad(loss, [a, b])):
        assert torch.equal(x, y)


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_peaked_rows(dtype, keep, monkeypatch):
    """Upstream gradients far from 1, and rows whose probabilities span all of
    fp32's exponents."""
    _keep(monkeypatch, keep)
    h, w, t = _operands(140, 64, 700, TYPES[dtype], spread=60.0)
    spread = torch.linspace(-60, 60, 140, device=DEV).exp2()   # from row to row
    for factor in (None, 2.0 ** -40, 2.0 ** 40, spread):
        if dtype == "f16" and factor is not None:
            continue   # (the gradients are no fp16 numbers)
        up = _upstream(140, "none") * (1.0 if factor is None else factor)
        got = _run(linear_cross_entropy, h, w, up, t, reduction="none")
        assert_head("upstream", got, h, w, up, "none", TYPES[dtype], targets=t)


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_pieces_of_the_vocabulary(dtype, keep, monkeypatch):
    """More than 256 MB of the logits' gradient: the backward in two pieces, the
    second a short one."""
    _keep(monkeypatch, keep)
    rows, dim, vocab = (2048, 64, 66001) if dtype != "f32" else (2048, 64, 33001)
    print(f"[case] pieces {dtype}", flush=True)
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    t[:4] = torch.tensor([vocab - 1, vocab - 2, 0, vocab // 2])
    up = _upstream(rows, "mean")
    got = _run(linear_cross_entropy, h, w, up, t)
    assert_head("pieces", got, h, w, up, "mean", TYPES[dtype], targets=t)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_gradient_only(dtype):
    """A frozen head, or hidden states that need no gradient: the other gradient
    is the same bit for bit."""
    h, w, t = _operands(130, 64, 500, TYPES[dtype])
    both = _run(linear_cross_entropy, h, w, torch.ones((), device=DEV), t)
    a = h.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(a, w, t), [a])[0], both[1])
    b = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(h, b, t), [b])[0], both[2])


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(33, 1096, 1), (33, 2056, 131), (65, 1032, 1001),
                                            (130, 2048, 258), (257, 1544, 515)])
def test_few_tiles_of_long_sums(rows, dim, vocab, dtype, keep, monkeypatch):
    """Products cut up in k, the sums of exponentials from the logits in memory."""
    print(f"[case] few tiles {dtype} {rows}x{dim}x{vocab}", flush=True)
    _keep(monkeypatch, keep)
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    up = _upstream(rows, "none")
    got = _run(linear_cross_entropy, h, w, up, t, reduction="none")
    assert_head("xent", got, h, w, up, "none", TYPES[dtype], targets=t)
    values, ids = _words(rows, vocab, 3)
    up = _upstream(rows, "mean")
    got = _run(linear_distill_loss, h, w, up, values, ids, temperature=2.0)
    assert_head("distill", got, h, w, up, "mean", TYPES[dtype], words=(values, ids, 2.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(2050, 72, 300), (4100, 264, 70)])
def test_weight_gradient_of_many_rows(rows, dim, vocab, dtype):
    """Few tiles of the weight's gradient, cut up in the rows."""
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    up = _upstream(rows, "sum")
    got = _run(linear_cross_entropy, h, w, up, t, reduction="sum")
    assert_head("rows", got, h, w, up, "sum", TYPES[dtype], targets=t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [512, 513])
def test_rows_on_both_sides_of_a_block_each(rows, dtype):
    h, w, t = _operands(rows, 264, 20000, TYPES[dtype])
    up = _upstream(rows, "none")
    got = _run(linear_cross_entropy, h, w, up, t, reduction="none")
    assert_head("rows", got, h, w, up, "none", TYPES[dtype], targets=t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 5, 66, 100])
def test_any_width(dim, dtype):
    """Widths whose rows are no whole 16-byte accesses."""
    h, w, t = _operands(40, dim, 130, TYPES[dtype])
    up = _upstream(40, "mean")
    got = _run(linear_cross_entropy, h, w, up, t)
    assert got[1].is_contiguous() and got[2].is_contiguous()
    assert_head("width", got, h, w, up, "mean", TYPES[dtype], targets=t)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    """Column slices, transposed, expanded and misaligned operands."""
    rows, dim, vocab = 70, 64, 300
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    up = _upstream(rows, "mean")
    want = _run(linear_cross_entropy, h, w, up, t)
    wide = torch.randn(rows, 3 * dim, device=DEV).to(TYPES[dtype])
    wide[:, dim:2 * dim] = h
    off = torch.empty(rows * dim + 1, device=DEV, dtype=TYPES[dtype])[1:].view(rows, dim)
    off.copy_(h)
    woff = torch.empty(vocab * dim + 1, device=DEV, dtype=TYPES[dtype])[1:].view(vocab, dim)
    woff.copy_(w)
    for a, b in ((wide[:, dim:2 * dim], w), (h.t().contiguous().t(), w.t().contiguous().t()),
                 (off, woff)):
        got = _run(linear_cross_entropy, a, b, up, t)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    one = h[:1].expand(rows, dim)
    base = h[:1].detach().requires_grad_()
    loss = linear_cross_entropy(base.expand(rows, dim), w, t)
    g = torch.autograd.grad(loss, [base])[0]
    full = _run(linear_cross_entropy, one.contiguous(), w, torch.ones((), device=DEV), t)
    assert torch.equal(loss.detach(), full[0])
    assert torch.equal(g, full[1].sum(0, keepdim=True))


def test_leading_dimensions_and_target_types():
    h, w, t = _operands(60, 64, 200, F32)
    want = linear_cross_entropy(h, w, t, reduction="none")
    got = linear_cross_entropy(h.view(4, 15, 64), w, t.view(4, 15).int(), reduction="none")
    assert got.shape == (4, 15) and torch.equal(got.view(-1), want)
    one = linear_cross_entropy(h[7], w, t[7], reduction="none")
    assert one.shape == () and abs(float(one) - float(want[7])) <= 1e-5
    values, ids = _words(60, 200, 8)
    want = linear_distill_loss(h, w, values, ids, reduction="none")
    got = linear_distill_loss(h.view(3, 20, 64), w, values.bfloat16().float().view(3, 20, 8),
                              ids.view(3, 20, 8).int(), reduction="none")
    assert got.shape == (3, 20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 40])
def test_rows_that_do_not_count(rows, dtype):
    """Ignored rows that hold NaN or infinities: nothing of them reaches the loss
    or the gradients, and theirs are zeros. All rows ignored: as the framework's
    mean, a loss of NaN and zeros. (In fp32 a wave that meets NaN or infinities
    computes its part of the tile again with fp32 products, whose sums round
    otherwise: the rows beside such a row stay within the bound, not the bit.)"""
    h, w, t = _operands(rows, 64, 300, TYPES[dtype])
    t[1], t[2] = -100, -100
    clean = h.clone()
    h[1], h[2, 3] = float("nan"), float("inf")
    clean[1:3] = 0
    for reduction in ("mean", "sum", "none"):
        up = _upstream(rows, reduction)
        got = _run(linear_cross_entropy, h, w, up, t, reduction=reduction)
        want = _run(linear_cross_entropy, clean, w, up, t, reduction=reduction)
        assert_head("rows", got, clean, w, up, reduction, TYPES[dtype], targets=t)
        for x, y in zip(got, want):
            assert dtype == "f32" or torch.equal(x, y)
        assert (got[1][1:3] == 0).all()
    got = _run(linear_cross_entropy, h, w, torch.ones((), device=DEV), torch.full_like(t, -100))
    assert torch.isnan(got[0]) and (got[1] == 0).all() and (got[2] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_rows_that_do_not_count(dtype):
    h, w, _ = _operands(40, 64, 300, TYPES[dtype])
    values, ids = _words(40, 300, 6)
    clean = h.clone()
    h[1], h[2] = float("nan"), float("inf")     # the empty rows of _words
    clean[1:3] = 0
    up = _upstream(40, "none")
    got = _run(linear_distill_loss, h, w, up, values, ids, temperature=2.0, reduction="none")
    want = _run(linear_distill_loss, clean, w, up, values, ids, temperature=2.0, reduction="none")
    assert_head("rows", got, clean, w, up, "none", TYPES[dtype], words=(values, ids, 2.0))
    for x, y in zip(got, want):
        assert dtype == "f32" or torch.equal(x, y)
    assert (got[0][1:3] == 0).all() and (got[1][1:3] == 0).all()
    got = _run(linear_distill_loss, h, w, torch.ones((), device=DEV), values,
               torch.full_like(ids, -1))
    assert torch.isnan(got[0]) and (got[1] == 0).all() and (got[2] == 0).all()


@pytest.mark.parametrize("rows", [4, 60])
def test_bad_words_make_the_row_nan(rows):
    h, w, t = _operands(rows, 64, 300, F32)
    t[:] = 5
    t[1], t[2] = 300, -7
    loss = linear_cross_entropy(h, w, t, reduction="none")
    assert torch.isnan(loss[1:3]).all() and torch.isfinite(loss[:1]).all() \
        and torch.isfinite(loss[3:]).all()
    values, ids = torch.zeros(rows, 2, device=DEV), torch.zeros(rows, 2, device=DEV).long()
    ids[1, 1], ids[2, 0] = 300, 1 << 40
    loss = linear_distill_loss(h, w, values, ids, reduction="none")
    assert torch.isnan(loss[1:3]).all() and torch.isfinite(loss[:1]).all() \
        and torch.isfinite(loss[3:]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_equal_logits(dtype):
    """Logits of hundreds (their exponentials overflow without the maximum), and
    logits that are all alike."""
    h, w, t = _operands(140, 64, 700, TYPES[dtype], spread=100.0)
    up = _upstream(140, "sum")
    got = _run(linear_cross_entropy, h, w, up, t, reduction="sum")
    assert_head("large", got, h, w, up, "sum", TYPES[dtype], targets=t)
    w = torch.zeros_like(w)
    got = _run(linear_cross_entropy, h, w, up, t, reduction="sum")
    assert_head("equal", got, h, w, up, "sum", TYPES[dtype], targets=t)


@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logits_of_minus_infinity(rows, dtype):
    """Words whose logit is -inf: probability 0, the rest as without them."""
    vocab, dim = 300, 64
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    h[:, 0] = 1.0
    w[:, 0] = 0.0
    t = t.clamp(max=199)
    want = linear_cross_entropy(h, w[:200], t, reduction="none")
    w[200:] = 0.0
    w[200:, 0] = float("-inf")
    got = linear_cross_entropy(h, w, t, reduction="none")
    assert torch.isfinite(got).all()
    assert_within("minus infinity", got, want, 2.0 ** -16 + 2.0 ** -20 * want.double().abs())
    up = torch.ones((), device=DEV)
    b = w.detach().requires_grad_()
    g = torch.autograd.grad(linear_cross_entropy(h, b, t), [b], up)[0]
    assert torch.isfinite(g).all() and (g[200:] == 0).all()


def test_small_upstream_gradients_in_fp16():
    """An fp16 gradient of the logits would vanish: 1 / 8192 of a probability."""
    h, w, t = _operands(200, 64, 5000, F16, spread=0.5)
    up = torch.full((), 3e-6, device=DEV)
    got = _run(linear_cross_entropy, h, w, up, t, reduction="sum")
    assert_head("small", got, h, w, up, "sum", F16, targets=t)
    up = 10.0 ** torch.linspace(-6, 2, 200, device=DEV)
    got = _run(linear_cross_entropy, h, w, up, t, reduction="none")
    assert_head("spread", got, h, w, up, "none", F16, targets=t)


def test_no_rows():
    _, w, _ = _operands(1, 64, 100, BF16)
    h = torch.empty(0, 64, device=DEV, dtype=BF16)
    t = torch.empty(0, dtype=torch.int64, device=DEV)
    got = _run(linear_cross_entropy, h, w, torch.ones((), device=DEV), t)
    assert torch.isnan(got[0]) and got[1].shape == (0, 64) and (got[2] == 0).all()
    assert float(linear_cross_entropy(h, w, t, reduction="sum")) == 0.0
    assert linear_cross_entropy(h, w, t, reduction="none").shape == (0,)
    ids = torch.empty(0, 4, dtype=torch.int64, device=DEV)
    got = _run(linear_distill_loss, h, w, torch.ones((), device=DEV), ids.float(), ids)
    assert torch.isnan(got[0]) and (got[2] == 0).all()


@pytest.mark.parametrize("rows", [8192, 8193, 16384, 16385, 20000])
def test_many_rows_of_losses(rows):
    """On both sides of the loss's one block."""
    h, w, t = _operands(rows, 8, 5, F32)
    up = _upstream(rows, "mean")
    got = _run(linear_cross_entropy, h, w, up, t)
    assert_head("rows", got, h, w, up, "mean", F32, targets=t)


@pytest.mark.parametrize("dtype", TYPES)
def test_bitwise_reproducible(dtype):
    h, w, t = _operands(400, 128, 4000, TYPES[dtype])
    values, ids = _words(400, 4000, 16)
    up = torch.ones((), device=DEV)
    for f, args in ((linear_cross_entropy, (t,)), (linear_distill_loss, (values, ids))):
        a, b = _run(f, h, w, up, *args), _run(f, h, w, up, *args)
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_gradients_against_differences():
    """Central differences of the fp32 loss along random directions: the
    truncation is below 2e-5 of the gradient there (step 1e-2 of unit-scale
    logits: h^2 / 6 of the third derivative), the rounding 2^-22 |loss| / step."""
    h, w, t = _operands(50, 64, 300, F32, spread=1.0)
    values, ids = _words(50, 300, 8)
    up = torch.ones((), device=DEV)
    g = _gen(9)
    for f, args in ((linear_cross_entropy, (t,)), (linear_distill_loss, (values, ids))):
        loss, dh, dw = _run(f, h, w, up, *args, reduction="sum")
        for x, grad, which in ((h, dh, 0), (w, dw, 1)):
            d = torch.randn(x.shape, generator=g, device=DEV)
            d = d / d.norm() * 0.1
            ends = []
            for s in (1.0, -1.0):
                y = x + s * d
                ends.append(float(f(*((y, w) if which == 0 else (h, y)), *args,
                                    reduction="sum").double()))
            want = float((grad.double() * d.double()).sum())
            slack = 2 * 2.0 ** -22 * abs(float(loss)) * 50 ** 0.5 + 2e-3 * float(d.norm()) ** 2
            assert abs((ends[0] - ends[1]) / 2 - want) <= slack + 1e-3 * abs(want), (ends, want)


def test_autocast_takes_its_type():
    h, w, t = _operands(64, 64, 300, F32)
    want = linear_cross_entropy(h.bfloat16(), w.bfloat16(), t)
    a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
    with torch.autocast("cuda", dtype=BF16):
        loss = linear_cross_entropy(a, b, t)
    assert torch.equal(loss.detach(), want)
    ga, gb = torch.autograd.grad(loss, [a, b])
    assert ga.dtype == F32 and gb.dtype == F32


def test_twice_differentiating_raises():
    h, w, t = _operands(8, 64, 50, F32)
    values, ids = _words(8, 50, 3)
    h.requires_grad_()
    for loss in (linear_cross_entropy(h, w, t), linear_distill_loss(h, w, values, ids)):
        with pytest.raises(HipScanError, match="once differentiable"):
            torch.autograd.grad(loss, [h], create_graph=True)


def test_compiled():
    h, w, t = _operands(40, 64, 300, BF16)
    values, ids = _words(40, 300, 4)

    def both(a, b):
        loss = linear_cross_entropy(a, b, t) + linear_distill_loss(a, b, values, ids)
        return loss, *torch.autograd.grad(loss, [a, b])

    def traced(a, b):
        return linear_cross_entropy(a, b, t) + linear_distill_loss(a, b, values, ids)

    h.requires_grad_()
    w.requires_grad_()
    want = both(h, w)
    loss = torch.compile(traced, backend="aot_eager")(h, w)
    got = (loss, *torch.autograd.grad(loss, [h, w]))
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_on_another_stream_and_captured():
    """On a side stream, and replayed from a graph with other data, eager work
    between the replays."""
    rows, dim, vocab = 150, 64, 700
    for dtype in (F32, BF16):
        sets = [_operands(rows, dim, vocab, dtype, seed=i) for i in range(4)]
        up = torch.ones((), device=DEV)
        want = [_run(linear_cross_entropy, *s[:2], up, s[2]) for s in sets]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _run(linear_cross_entropy, *sets[0][:2], up, sets[0][2])
        torch.cuda.current_stream().wait_stream(side)
        for x, y in zip(got, want[0]):
            assert torch.equal(x, y)
        h, w, t = (x.clone() for x in sets[0])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                _run(linear_cross_entropy, h, w, up, t)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _run(linear_cross_entropy, h, w, up, t)
        for s, ref in zip(sets, want):
            for x, y in zip((h, w, t), s):
                x.copy_(y)
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(out, ref):
                assert torch.equal(x, y)
            _run(linear_cross_entropy, *sets[1][:2], up, sets[1][2])
            torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_two_calls_at_once(dtype):
    """Two threads, each on a stream of its own, with operands of their own."""
    from concurrent.futures import ThreadPoolExecutor
    sets = [_operands(rows, 128, vocab, TYPES[dtype], seed=rows)
            for rows, vocab in ((40, 3000), (300, 1100))]
    up = torch.ones((), device=DEV)
    want = [_run(linear_cross_entropy, h, w, up, t) for h, w, t in sets]
    torch.cuda.synchronize()

    def work(i):
        h, w, t = sets[i]
        stream = torch.cuda.Stream()
        out = []
        with torch.cuda.stream(stream):
            for _ in range(10):
                out.append(_run(linear_cross_entropy, h, w, up, t))
        stream.synchronize()
        return out
    with ThreadPoolExecutor(2) as pool:
        for i, out in enumerate(pool.map(work, range(2))):
            for got in out:
                assert all(torch.equal(x, y) for x, y in zip(got, want[i]))


def test_op_argument_errors():
    h, w, t = _operands(8, 64, 50, BF16)
    ops = torch.ops.mamba_hip
    with pytest.raises(HipScanError, match="16-byte"):
        ops.linear_xent_fwd(h[:, :60], w[:, :60], t, -100, 1)
    with pytest.raises(HipScanError, match="must both be"):
        ops.linear_xent_fwd(h.float(), w, t, -100, 1)
    with pytest.raises(HipScanError, match="int64"):
        ops.linear_xent_fwd(h, w, t.int(), -100, 1)
    with pytest.raises(HipScanError, match="reduction"):
        ops.linear_xent_fwd(h, w, t, -100, 3)
    loss, saved = ops.linear_xent_fwd(h, w, t, -100, 1)
    with pytest.raises(HipScanError, match="saved"):
        ops.linear_xent_bwd(torch.ones((), device=DEV), h, w, t, saved[:-1], 1, True, True)
    with pytest.raises(HipScanError, match="grad"):
        ops.linear_xent_bwd(torch.ones(8, device=DEV), h, w, t, saved, 1, True, True)
    loss, saved = ops.linear_xent_fwd(h, w, t, -100, 1, True)
    off = torch.empty(saved.numel() + 1, device=DEV)[1:]
    with pytest.raises(HipScanError, match="aligned"):
        ops.linear_xent_bwd(torch.ones((), device=DEV), h, w, t, off, 1, True, True)
    values, ids = _words(8, 50, 4)
    with pytest.raises(HipScanError, match="int64"):
        ops.linear_distill_fwd(h, w, values, ids.int(), 1.0, 1)
    with pytest.raises(HipScanError, match="temperature"):
        ops.linear_distill_fwd(h, w, values, ids, 0.0, 1)
    with pytest.raises(HipScanError, match="teacher_logits"):
        ops.linear_distill_fwd(h, w, values[:, :3].contiguous(), ids, 1.0, 1)


@pytest.mark.parametrize("rows,dtype,keep", [(4, "bf16", True), (40, "bf16", False),
                                             (40, "bf16", True), (4, "f32", False)])
def test_weights_past_32_bits(rows, dtype, keep, monkeypatch):
    """A weight of more than 2^31 elements whose words but the last 1000 are out of
    reach (their probabilities are 0 exactly): the small weight's results."""
    print(f"[case] large weight {rows} {dtype} {keep}", flush=True)
    _keep(monkeypatch, keep)
    dim, vocab, last = 1032, (1 << 21) + 3, 1000
    h, w, t = _operands(rows, dim, last, TYPES[dtype])
    h[:, 0], w[:, 0] = 1.0, 0.0
    up = _upstream(rows, "none")
    want = _run(linear_cross_entropy, h, w, up, t, reduction="none")
    large = torch.zeros(vocab, dim, dtype=TYPES[dtype], device=DEV)
    large[:, 0] = -1024.0
    large[-last:] = w
    got = _run(linear_cross_entropy, h, large, up, torch.where(t < 0, t, t + vocab - last),
               reduction="none")
    assert (got[2][:-last] == 0).all()
    # The sums' order differs: of the logits by the small bound, dh's by its rounding.
    z = sum_error(dim) * (h.double().abs() @ w.double().abs().t())
    p = 2 * z.amax(1) + 2.0 ** -16
    assert_within("loss", got[0], want[0], p + 2.0 ** -20 * want[0].double().abs())
    unit = 2 * max(UNIT[TYPES[dtype]], 2.0 ** -20)
    dz = up.double().abs()[:, None] * (2 * p[:, None] + unit) * torch.ones_like(z)
    assert_within("dW", got[2][-last:], want[2],
                  dz.t() @ h.double().abs() + unit * want[2].double().abs())
    z = h.double() @ w.double().t()
    q = z.softmax(1)
    q[torch.arange(rows, device=DEV), t.clamp(min=0)] += 1.0
    assert_within("dh", got[1], want[1], (q * dz) @ w.double().abs()
                  + unit * want[1].double().abs())


def test_matches_the_logits_loss():
    """The same loss as the package's cross_entropy of the logits."""
    from mamba_metal_scan_amd import cross_entropy
    h, w, t = _operands(200, 64, 1000, F32)
    a = linear_cross_entropy(h, w, t)
    b = cross_entropy(F.linear(h, w), t)
    assert abs(float(a) - float(b)) <= 1e-5 * abs(float(b))
