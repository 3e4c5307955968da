"""GPU parity of the distillation of given logits with 64 bits: any vocabulary,
type, row stride and alignment, rows and words that do not count. Bounds:
head_reference.py, the logits being exact."""
from __future__ import annotations

import math

import pytest
import torch

from head_reference import Reference, UNIT, assert_within
from mamba_metal_scan_amd import distill_loss
from mamba_metal_scan_amd._native import HipScanError

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (1 << 31))


def _case(rows, vocab, k, dtype, seed=0, spread=3.0):
    g = _gen(rows, vocab, k, seed)
    z = (spread * torch.randn(rows, vocab, generator=g, device=DEV)).to(dtype)
    ids = torch.rand(rows, max(vocab, k), generator=g, device=DEV).argsort(1)[:, :k] % vocab
    values = 2.0 * torch.randn(rows, k, generator=g, device=DEV)
    keep = torch.rand(rows, k, generator=g, device=DEV) < 0.6
    some = torch.rand(rows, 1, generator=g, device=DEV) < 0.33
    ids = torch.where(some & ~keep, -1, ids)
    if rows > 2:
        ids[1] = -1
        values[2] = -math.inf
        ids[0, 0] = vocab - 1
        if k > 1:
            ids[0, 1] = ids[0, 0]
            values[0, -1] = -math.inf
    return z, values, ids


def _run(z, values, ids, up, **kw):
    z = z.detach().requires_grad_()
    loss = distill_loss(z, values, ids, **kw)
    return loss.detach(), *torch.autograd.grad(loss, [z], up)


def _check(name, got, z, values, ids, temperature, up, reduction, dtype):
    zd = z.double()
    # z / t: its product with log2(e) / t (two roundings) and the exponent's fma
    zerr = 2.0 ** -22 * zd.abs()
    ref = Reference(zd, zerr, words=(values, ids, temperature), unit=UNIT[dtype])
    loss, err, share = ref.reduced(reduction)
    assert_within(name + " loss", got[0], loss, err + 1e-30)
    u = up.double() * share
    u = u[:, None] if u.dim() else u
    err = ref.dz_err * u.abs() + 2.0 ** -21 * (ref.dz * u).abs() + SMALLEST[dtype]
    assert_within(name + " dlogits", got[1], ref.dz * u, err)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,k,temperature",
                         [(1, 1, 1, 1.0), (3, 7, 3, 2.0), (8, 1001, 5, 1.0), (5, 4096, 64, 4.0),
                          (4, 50257, 1000, 0.5), (33, 2049, 20, 1.5), (2, 100003, 128, 2.0)])
def test_matches_64_bits(rows, vocab, k, temperature, dtype):
    print(f"[case] distill {dtype} {rows}x{vocab} k {k}", flush=True)
    z, values, ids = _case(rows, vocab, k, TYPES[dtype])
    for reduction in ("mean", "sum", "none"):
        up = torch.randn((rows,) if reduction == "none" else (), generator=_gen(rows, 5),
                         device=DEV)
        got = _run(z, values, ids, up, temperature=temperature, reduction=reduction)
        _check(reduction, got, z, values, ids, temperature, up, reduction, TYPES[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [5, 8, 15, 16, 17, 1023, 2050])
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_rows_of_any_length_and_alignment(vocab, offset, dtype):
    rows = 6
    z, values, ids = _case(rows, vocab, 4, TYPES[dtype])
    buf = torch.empty(rows * vocab + offset, device=DEV, dtype=TYPES[dtype])
    view = buf[offset:].view(rows, vocab)
    view.copy_(z)
    up = torch.ones((), device=DEV)
    got = _run(view, values, ids, up)
    _check("offset", got, z, values, ids, 1.0, up, "mean", TYPES[dtype])
    wide = torch.zeros(rows, vocab + 3 + offset, device=DEV, dtype=TYPES[dtype])
    wide[:, offset:offset + vocab] = z
    got2 = _run(wide[:, offset:offset + vocab], values, ids, up)
    _check("slice", got2, z, values, ids, 1.0, up, "mean", TYPES[dtype])
    got3 = _run(z.t().contiguous().t(), values, ids, up)
    _check("transposed", got3, z, values, ids, 1.0, up, "mean", TYPES[dtype])


def test_logits_past_32_bits():
    """More than 2^31 logits: the last rows against 64 bits."""
    rows, vocab, last = 66000, 32769, 50
    z, values, ids = _case(last, vocab, 20, torch.bfloat16)
    large = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=DEV)
    large[-last:] = z
    all_ids = torch.zeros(rows, 20, dtype=torch.int64, device=DEV)
    all_ids[-last:] = ids
    all_values = torch.zeros(rows, 20, device=DEV)
    all_values[-last:] = values
    up = torch.randn(rows, generator=_gen(3), device=DEV)
    got = _run(large, all_values, all_ids, up, temperature=2.0, reduction="none")
    # (Not bit for bit a small call's: a row's sums begin at its first 16-byte boundary,
    # and its first element lies (rows - last) 32769 mod 8 = 6 elements off one here.)
    _check("last rows", (got[0][-last:], got[1][-last:]), z, values, ids, 2.0, up[-last:], "none",
           torch.bfloat16)


def test_large_and_masked_logits():
    z, values, ids = _case(20, 3000, 8, torch.float32, spread=100.0)
    up = torch.ones((), device=DEV)
    got = _run(z, values, ids, up, temperature=2.0)
    _check("large", got, z, values, ids, 2.0, up, "mean", torch.float32)
    z = torch.randn(6, 3000, device=DEV)
    z[:, 2000:] = -math.inf
    z[:, 1000:1500] = torch.finfo(torch.float32).min
    values, ids = torch.randn(6, 4, device=DEV), torch.arange(24, device=DEV).view(6, 4)
    got = _run(z, values, ids, up)
    want = _run(z[:, torch.cat([torch.arange(1000), torch.arange(1500, 2000)]).to(DEV)]
                .contiguous(), values, ids, up)
    assert torch.isfinite(got[0]) and torch.isfinite(got[1]).all()
    assert abs(float(got[0]) - float(want[0])) <= 2.0 ** -16 * (1 + abs(float(want[0])))
    assert (got[1][:, 2000:] == 0).all() and (got[1][:, 1000:1500] == 0).all()


def test_a_word_that_the_student_rules_out():
    """A word of the teacher with a logit of -inf: an infinite loss, and the
    gradient of the row's formula; with probability 0 it counts for nothing."""
    z = torch.randn(2, 100, device=DEV)
    z[:, 7] = -math.inf
    values = torch.tensor([[0.0, 0.0], [0.0, -math.inf]], device=DEV)
    ids = torch.tensor([[3, 7], [3, 7]], device=DEV)
    got = _run(z, values, ids, torch.ones(2, device=DEV), reduction="none")
    assert got[0][0] == math.inf and torch.isfinite(got[0][1])
    assert torch.isfinite(got[1]).all() and abs(float(got[1][0, 7]) + 0.5) <= 1e-6
    assert got[1][1, 7] == 0


def test_bad_words_and_values():
    z = torch.randn(5, 50, device=DEV)
    values, ids = torch.zeros(5, 2, device=DEV), torch.zeros(5, 2, device=DEV).long()
    ids[1, 1] = 50
    ids[2, 0] = 1 << 40
    values[3, 0] = math.nan
    loss = distill_loss(z, values, ids, reduction="none")
    assert torch.isnan(loss[1:4]).all() and torch.isfinite(loss[[0, 4]]).all()


def test_empty_and_no_rows():
    z, values, ids = _case(6, 300, 4, torch.float32)
    z[1], z[2] = math.nan, math.inf
    up = torch.ones(6, device=DEV)
    got = _run(z, values, ids, up, reduction="none")
    assert (got[0][1:3] == 0).all() and (got[1][1:3] == 0).all()
    got = _run(z, values, torch.full_like(ids, -5), torch.ones((), device=DEV))
    assert torch.isnan(got[0]) and (got[1] == 0).all()
    got = _run(z[:0], values[:0], ids[:0], torch.ones((), device=DEV))
    assert torch.isnan(got[0]) and got[1].shape == (0, 300)
    assert float(distill_loss(z[:0], values[:0], ids[:0], reduction="sum")) == 0


def test_leading_dimensions_and_types():
    z, values, ids = _case(12, 100, 4, torch.bfloat16)
    want = distill_loss(z, values.bfloat16().float(), ids, reduction="none")
    got = distill_loss(z.view(3, 4, 100), values.bfloat16().view(3, 4, 4),
                       ids.int().view(3, 4, 4), reduction="none")
    assert got.shape == (3, 4) and torch.equal(got.view(-1), want)
    one = distill_loss(z[5], values[5], ids[5], reduction="none")
    assert one.shape == ()


def test_gradients_against_differences():
    """Along random directions; the loss's third derivative is below 1 per unit
    step cubed and row, the rounding 2^-22 of the loss."""
    z, values, ids = _case(20, 200, 8, torch.float32, spread=1.0)
    loss, g = _run(z, values, ids, torch.ones((), device=DEV), temperature=2.0, reduction="sum")
    for seed in range(3):
        d = torch.randn(z.shape, generator=_gen(seed), device=DEV)
        d = d / d.norm() * 0.2
        ends = [float(distill_loss(z + s * d, values, ids, temperature=2.0, reduction="sum"))
                for s in (1.0, -1.0)]
        want = float((g.double() * d.double()).sum())
        assert abs((ends[0] - ends[1]) / 2 - want) <= 0.2 ** 3 / 6 + 2.0 ** -21 * abs(float(loss))


def test_reproducible_streams_and_graphs():
    sets = [_case(40, 3001, 16, torch.bfloat16, seed=i) for i in range(3)]
    up = torch.ones((), device=DEV)
    want = [_run(*s, up, temperature=2.0) for s in sets]
    again = _run(*sets[0], up, temperature=2.0)
    assert all(torch.equal(x, y) for x, y in zip(want[0], again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    z, values, ids = (x.clone() for x in sets[0])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = _run(z, values, ids, up, temperature=2.0)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want[0], got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(z, values, ids, up, temperature=2.0)
    for s, ref in zip(sets, want):
        for x, y in zip((z, values, ids), s):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, ref))
        _run(*sets[1], up, temperature=2.0)
        torch.cuda.synchronize()


def test_op_argument_errors():
    z, values, ids = _case(4, 50, 3, torch.float32)
    ops = torch.ops.mamba_hip
    with pytest.raises(HipScanError, match="float32, bfloat16"):
        ops.distill_fwd(z.double(), values, ids, 1.0, 1)
    with pytest.raises(HipScanError, match="int64"):
        ops.distill_fwd(z, values, ids.int(), 1.0, 1)
    with pytest.raises(HipScanError, match="contiguous rows"):
        ops.distill_fwd(z.t(), values.repeat(13, 1)[:50].contiguous(),
                        ids.repeat(13, 1)[:50].contiguous(), 1.0, 1)
    with pytest.raises(HipScanError, match="k in"):
        ops.distill_fwd(z, torch.zeros(4, 1025, device=DEV),
                        torch.zeros(4, 1025, dtype=torch.int64, device=DEV), 1.0, 1)
    loss, saved = ops.distill_fwd(z, values, ids, 1.0, 1)
    with pytest.raises(HipScanError, match="saved"):
        ops.distill_bwd(torch.ones((), device=DEV), z, ids, saved[:-1], 1.0, 1)
    z.requires_grad_()
    with pytest.raises(HipScanError, match="once differentiable"):
        torch.autograd.grad(distill_loss(z, values, ids), [z], create_graph=True)
