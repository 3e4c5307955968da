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


@pytest.mark.parametrize("dtype", TYPES)
def test_compiled_in_one_graph(dtype):
    """torch.compile with fullgraph at several row counts, odd widths and unaligned
    views: bit for bit the eager losses and gradients (in fp32, whose logits eager keeps
    from a limit on, the same rule applies to both)."""
    print(f"[case] compiled {dtype}", flush=True)

    def losses(a, b, t, values, ids):
        return (linear_cross_entropy(a, b, t),
                linear_distill_loss(a, b, values, ids, temperature=2.0, reduction="none"),
                distill_loss(a @ b.t(), values, ids))
    torch._dynamo.reset()
    f = torch.compile(losses, backend="aot_eager", fullgraph=True)
    for rows, dim in ((40, 64), (3, 64), (300, 64), (40, 50)):
        h, w, t = _operands(rows, dim, 301, TYPES[dtype])
        ids = torch.randint(0, 301, (rows, 4), generator=_gen(rows), device=DEV)
        values = torch.randn(rows, 4, generator=_gen(rows, 1), device=DEV)
        off = torch.empty(h.numel() + 1, dtype=h.dtype, device=DEV)[1:].view(rows, dim)
        off.copy_(h)
        for a in (h, off):
            results = []
            for fn in (losses, f):
                x, y = a.detach().requires_grad_(), w.detach().requires_grad_()
                out = fn(x, y, t, values, ids)
                up = [torch.ones_like(o) for o in out]
                results.append((*(o.detach() for o in out),
                                *torch.autograd.grad(out, [x, y], up)))
            for one, two in zip(*results):
                assert torch.equal(one, two)
    torch._dynamo.reset()


def test_compiled_model_losses():
    from mamba_metal_scan_amd import MambaConfig, TinyMamba
    torch.manual_seed(0)
    model = TinyMamba(MambaConfig(vocab_size=601, d_model=64, n_layers=2, d_ff=256,
                                  scan_impl="hip")).to(DEV)
    idx = torch.randint(0, 601, (3, 41), generator=_gen(3), device=DEV)
    x, t = idx[:, :-1].contiguous(), idx[:, 1:].contiguous()
    ids = torch.randint(0, 601, (3, 40, 5), generator=_gen(4), device=DEV)
    values = torch.randn(3, 40, 5, generator=_gen(5), device=DEV)

    def both():
        return model.loss(x, t) + model.distill(x, values, ids, temperature=2.0)
    torch._dynamo.reset()
    results = []
    for fn in (both, torch.compile(both, backend="aot_eager", fullgraph=True)):
        model.zero_grad(set_to_none=True)
        loss = fn()
        loss.backward()
        results.append((loss.detach(), [p.grad.clone() for p in model.parameters()]))
    torch._dynamo.reset()
    (l1, g1), (l2, g2) = results
    # (the bar of the compiled model's own test)
    assert abs(float(l1) - float(l2)) <= 1e-6 * float(l1)
    for a, b in zip(g1, g2):
        assert float((a - b).abs().max()) <= 1e-5 * max(1.0, float(a.abs().max()))


def test_the_model_passes_on_what_may_be_held():
    """logits_bytes through TinyMamba.loss and .distill: what is held until the backward
    grows by the logits where they may be kept, the gradients stay."""
    from mamba_metal_scan_amd import MambaConfig, TinyMamba
    torch.manual_seed(0)
    model = TinyMamba(MambaConfig(vocab_size=20000, d_model=64, n_layers=1, d_ff=256,
                                  scan_impl="hip")).to(DEV)
    x = torch.randint(0, 20000, (4, 100), generator=_gen(3), device=DEV)
    ids = torch.randint(0, 20000, (4, 100, 5), generator=_gen(4), device=DEV)
    values = torch.randn(4, 100, 5, generator=_gen(5), device=DEV)
    logits = 400 * 20000 * 4
    for f in (lambda **kw: model.loss(x, x, **kw),
              lambda **kw: model.distill(x, values, ids, 2.0, **kw)):
        held, grads = [], []
        for kw in ({"logits_bytes": 0}, {"logits_bytes": logits - 1}, {"logits_bytes": logits},
                   {}):
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            loss = f(**kw)
            held.append(torch.cuda.memory_allocated() - before)
            grads.append(torch.autograd.grad(loss, list(model.parameters())))
            del loss
        assert abs(held[1] - held[0]) < logits // 8
        for n in held[2:]:
            assert logits <= n - held[0] < logits + logits // 8
        for a, b in zip(grads[0], grads[2]):   # (fp32's bar of the model's other paths)
            assert float((a - b).abs().max()) <= 1e-4 * float(a.abs().max()) + 1e-9


def test_targets_of_any_shape():
    """Targets (B T,) beside tokens (B, T), which forward takes: both of loss's paths."""
    from mamba_metal_scan_amd import MambaConfig, TinyMamba
    torch.manual_seed(0)
    model = TinyMamba(MambaConfig(vocab_size=601, d_model=64, n_layers=1, d_ff=256,
                                  scan_impl="hip")).to(DEV)
    x = torch.randint(0, 601, (3, 40), generator=_gen(3), device=DEV)
    for _ in range(2):
        want = model.loss(x, x)
        assert torch.equal(model.loss(x, x.view(-1)), want)
        rows = model.loss(x, x.view(-1), reduction="none")
        assert rows.shape == (120,)
        assert torch.equal(rows.view(3, 40), model.loss(x, x, reduction="none"))
        with pytest.raises(ValueError):
            model.loss(x, x[:, :-1])
        model.head.register_forward_hook(lambda m, a, o: None)   # then the logits' loss


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(4, 64, 900), (40, 1032, 301), (300, 64, 1300)])
def test_captured_together(rows, dim, vocab, dtype):
    """The three losses and their gradients in one graph, replayed with other data (rows
    that do not count, a row of one value), eager work between the replays."""
    print(f"[case] captured {dtype} {rows}x{dim}x{vocab}", flush=True)
    dt = TYPES[dtype]

    def data(seed):
        h, w, t = _operands(rows, dim, vocab, dt, seed)
        g = _gen(seed, rows)
        t[1] = -100
        ids = torch.randint(0, vocab, (rows, 4), generator=g, device=DEV)
        ids[2] = -1
        z = torch.randn(rows, vocab, generator=g, device=DEV).to(dt)
        z[seed % 3] = torch.finfo(dt).min
        return [h, w, t, ids, torch.randn(rows, 4, generator=g, device=DEV), z,
                torch.randn(rows, generator=g, device=DEV)]

    def run(h, w, t, ids, values, z, up):
        h, w, z = (x.detach().requires_grad_() for x in (h, w, z))
        losses = (linear_cross_entropy(h, w, t, reduction="none"),
                  linear_distill_loss(h, w, values, ids, temperature=2.0, reduction="none"),
                  distill_loss(z, values, ids, temperature=2.0, reduction="none"))
        out = [x.detach() for x in losses]
        out += torch.autograd.grad(losses[0], [h, w], up)
        out += torch.autograd.grad(losses[1], [h, w], up)
        return out + list(torch.autograd.grad(losses[2], [z], up))
    sets = [data(i) for i in range(4)]
    want = [run(*s) for s in sets]
    held = [x.clone() for x in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*held)
    for s, ref in zip(sets, want):
        for x, y in zip(held, s):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, ref):
            assert torch.equal(x, y)
        run(*sets[1])
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(3, 64, 130), (40, 64, 301), (33, 2056, 131),
                                            (595, 64, 2832)])
def test_logits_of_the_ids_are_those_of_the_sums(rows, dim, vocab, dtype):
    """Where the forward keeps its logits, the ids' are taken from them: dot products of
    their own would differ by the sums' rounding, which then does not cancel against the
    log-sum-exp's in rows that are sure of their word."""
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    k = 5
    ids = torch.randint(0, vocab, (rows, k), generator=_gen(rows), device=DEV)
    ids[0, 0] = -1
    ops = torch.ops.mamba_hip

    def logits(saved, n):
        n = (n + 3) // 4 * 4
        a, b = (vocab, rows) if dtype == "f32" else (rows, vocab)
        z = saved[n:].view(a, (b + 3) // 4 * 4)[:, :b]
        return z.t() if dtype == "f32" else z
    _, saved = ops.linear_xent_fwd(h, w, t, -100, 1, True)
    z = logits(saved, 4 + 4 * rows)
    assert torch.equal(saved[4 + 3 * rows:4 + 4 * rows], z.gather(1, t[:, None])[:, 0])
    _, saved = ops.linear_distill_fwd(h, w, torch.zeros(rows, k, device=DEV), ids, 1.0, 1, True)
    z = logits(saved, 4 + (3 + 2 * k) * rows)
    picked = saved[4 + 3 * rows:4 + (3 + k) * rows].view(rows, k)
    assert torch.equal(picked, torch.where(ids < 0, 0.0, z.gather(1, ids.clamp(min=0))))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_kept_logits_past_32_bits(dtype, monkeypatch):
    """More than 2^31 kept logits: the last rows' and words' gradients are those of
    logits formed again (the ids' logits are another sum there, 2^-17 of a probability
    by head_reference.py's bound of 64 terms; in bf16 they and the rest round once)."""
    from mamba_metal_scan_amd import _native
    print(f"[case] kept {dtype}", flush=True)
    rows, dim, vocab = 70001, 64, 33003
    h, w, t = _operands(rows, dim, vocab, TYPES[dtype])
    t[-7:] = vocab - 1 - torch.arange(7, device=DEV)
    up = torch.randn(rows, generator=_gen(2), device=DEV)
    got = []
    for keep in (True, False):
        monkeypatch.setattr(_native, "keeps_logits", lambda *a: keep)
        a, b = h.requires_grad_(), w.requires_grad_()
        loss = linear_cross_entropy(a, b, t, reduction="none")
        got.append((loss.detach(), *torch.autograd.grad(loss, [a, b], up)))
        torch.cuda.empty_cache()
    eps = torch.finfo(TYPES[dtype]).eps
    assert float((got[0][0] - got[1][0]).abs().max()) <= 2.0 ** -14
    rel = 2.0 ** -14 + (2 * eps if dtype == "bf16" else 0.0)
    for x, y in zip(got[0][1:], got[1][1:]):
        x, y = x.double(), y.double()
        for part in (slice(None), slice(-300, None)):
            assert float((x[part] - y[part]).norm()) <= rel * float(y[part].norm())
