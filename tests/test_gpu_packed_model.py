"""TinyMamba over packed sequences on the GPU: prefill, generation and training of packed documents
against the same sequences one by one; requests that come and go against a pool."""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from helpers import assert_close
from mamba_metal_scan_amd import (MambaConfig, TinyMamba, conv1d_silu, conv1d_silu_packed,
                                  conv1d_silu_step, sample_tokens, selective_scan,
                                  selective_scan_packed, selective_state_step_slots)

pytestmark = pytest.mark.gpu
LENS = [5, 1, 40, 17]


def _model(seed=0, **kw):
    torch.manual_seed(seed)
    cfg = MambaConfig(vocab_size=211, d_model=64, n_layers=3, d_ff=128, scan_impl="hip", **kw)
    return TinyMamba(cfg).cuda()


def _prompts(lens, vocab=211, seed=1):
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, vocab, (sum(lens),), generator=g).cuda()
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    return idx, cu, list(idx.split(lens))


def test_prefill_is_each_prompt_alone():
    model = _model()
    idx, cu, parts = _prompts(LENS)
    with torch.no_grad():
        cache = {}
        logits = model.prefill(idx, cu, cache)
        for s, p in enumerate(parts):
            own = {}
            want = model(p[None], cache=own)[0][0, -1]
            assert_close("logits", logits[s], want, 2e-5)
            for a, b in zip(cache["blocks"], own["blocks"]):
                assert_close("h", a["h"][s], b["h"][0], 2e-5)
                assert_close("conv", a["conv"][s], b["conv"][0], 2e-5)
        # the next token of all of them
        nxt = torch.tensor([[3], [7], [1], [9]], device="cuda")
        got = model(nxt, cache=cache)[0][:, -1]
        for s, p in enumerate(parts):
            want = model(torch.cat([p, nxt[s]])[None])[0][0, -1]
            assert_close("next", got[s], want, 5e-5)


def test_prefill_in_parts():
    model = _model()
    idx, cu, parts = _prompts([40, 23])
    with torch.no_grad():
        whole, split = {}, {}
        want = model.prefill(idx, cu, whole)
        first = torch.cat([parts[0][:16], parts[1][:1]])
        model.prefill(first, torch.tensor([0, 16, 17], device="cuda"), split)
        rest = torch.cat([parts[0][16:], parts[1][1:]])
        got = model.prefill(rest, torch.tensor([0, 24, 46], device="cuda"), split)
        assert_close("logits", got, want, 2e-5)
        for a, b in zip(split["blocks"], whole["blocks"]):
            assert_close("h", a["h"], b["h"], 2e-5)
    # a prompt of no token
    with torch.no_grad():
        out = model.prefill(idx[:4], torch.tensor([0, 0, 4], device="cuda"), {})
        assert torch.isnan(out[0]).all() and not torch.isnan(out[1]).any()


def test_generate_is_prefill_and_draws():
    model = _model()
    idx, cu, parts = _prompts(LENS)
    u = torch.rand(4, 6, device="cuda")
    settings = dict(temperature=torch.tensor([0.0, 0.7, 1.0, 1.3], device="cuda"), top_k=20,
                    top_p=0.95, min_p=0.0)
    got = model.generate(idx, cu, 6, uniform=u, **settings)
    assert got.shape == (4, 6) and got.dtype == torch.int64
    assert ((got >= 0) & (got < 211)).all()
    # each step's draw from the logits of all the tokens so far
    with torch.no_grad():
        for s, p in enumerate(parts):
            for i in range(6):
                logits = model(torch.cat([p, got[s, :i]])[None])[0][:, -1]
                own = dict(settings, temperature=settings["temperature"][s:s + 1])
                # (the token by token path's logits differ in their last bits: a number next
                # to a border may fall on either side of it)
                near = [int(sample_tokens(logits, (u[s:s + 1, i] + e).clamp(0, 1), **own))
                        for e in (-2e-4, 0.0, 2e-4)]
                assert int(got[s, i]) in near, (s, i)
    again = model.generate(idx, cu, 6, uniform=u, **settings)
    assert torch.equal(got, again)
    g1, g2 = (torch.Generator(device="cuda").manual_seed(5) for _ in range(2))
    assert torch.equal(model.generate(idx, cu, 3, generator=g1),
                       model.generate(idx, cu, 3, generator=g2))
    greedy = model.generate(idx, cu, 3, temperature=0.0)
    with torch.no_grad():
        for s, p in enumerate(parts):
            assert int(greedy[s, 0]) == int(model(p[None])[0][0, -1].argmax())
    assert model.generate(idx, cu, 0).shape == (4, 0)
    with pytest.raises(ValueError, match="uniform"):
        model.generate(idx, cu, 2, uniform=u)


@pytest.mark.parametrize("dtype", [None, torch.bfloat16])
def test_loss_of_packed_documents(dtype):
    """The sum over the tokens of all documents and its gradients, as of each alone."""
    model = _model()
    idx, cu, parts = _prompts(LENS)
    targets, _, tparts = _prompts(LENS, seed=9)
    with torch.autocast("cuda", dtype, enabled=dtype is not None):
        loss = model.loss(idx, targets, reduction="sum", cu_seqlens=cu)
        loss.backward()
        got = {n: p.grad.clone() for n, p in model.named_parameters()}
        model.zero_grad()
        want = sum(model.loss(p[None], t[None], reduction="sum")
                   for p, t in zip(parts, tparts))
        want.backward()
    bar = 5e-5 if dtype is None else 4e-2
    assert_close("loss", loss, want, bar)
    for n, p in model.named_parameters():
        assert_close(n, got[n], p.grad, bar)
    per_token = model.loss(idx, targets, reduction="none", cu_seqlens=cu)
    assert per_token.shape == targets.shape


def test_a_document_does_not_see_another():
    model = _model()
    idx, cu, _ = _prompts(LENS)
    targets, _, _ = _prompts(LENS, seed=3)
    with torch.no_grad():
        a = model.loss(idx, targets, reduction="none", cu_seqlens=cu)
        other = idx.clone()
        other[:6] = (other[:6] + 1) % 211
        b = model.loss(other, targets, reduction="none", cu_seqlens=cu)
    assert torch.equal(a[6:], b[6:]) and not torch.equal(a[:6], b[:6])


def test_packed_paths_refuse_the_torch_path():
    model = _model()
    idx, cu, _ = _prompts(LENS)
    with pytest.raises(RuntimeError, match="packed sequences"):
        model.prefill(idx[None], cu, {})
    plain = TinyMamba(MambaConfig(vocab_size=50, d_model=32, n_layers=1, scan_impl="torch"))
    with pytest.raises(RuntimeError, match="packed sequences"):
        plain.prefill(torch.zeros(3, dtype=torch.int64), torch.tensor([0, 3]), {})


def test_requests_that_come_and_go():
    """Packed prompts into a pool, tokens by slot, a request that leaves and one that takes its
    slot: every request's outputs as of its tokens alone through the rectangular path."""
    d, n, k, pool = 48, 16, 4, 6
    g = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    w, bias, aneg = randn(d, 1, k), randn(d), randn(d, n).exp()
    wb, wc, wdt = randn(d, n) / d ** 0.5, randn(d, n) / d ** 0.5, randn(d, d) / d ** 0.5

    def proj(x):
        return 0.001 + 0.099 * torch.sigmoid(x @ wdt), x @ wb, x @ wc

    def alone(x):   # (T, d) through the framework's rectangular operators
        xc = conv1d_silu(x[None], w, bias)
        dt, b, c = proj(xc)
        return selective_scan(xc, dt, aneg, b, c, impl="hip")[0]

    windows = torch.full((pool, d, k - 1), float("nan"), device="cuda")
    states = torch.full((pool, d, n), float("nan"), device="cuda")
    seen, outs = {}, {}

    def prompts(requests):   # {slot: length}, from nothing
        lens = list(requests.values())
        x = randn(sum(lens), d)
        cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
        xc, win = conv1d_silu_packed(x, w, bias, cu, return_window=True)
        dt, b, c = proj(xc)
        y, h = selective_scan_packed(xc, dt, aneg, b, c, cu, return_state=True)
        at = torch.tensor(list(requests), device="cuda")
        windows[at], states[at] = win, h
        for slot, xs, ys in zip(requests, x.split(lens), y.split(lens)):
            seen[slot], outs[slot] = [xs], [ys]

    def tokens(slots):       # one token each; -1: a row of a padded batch
        x = randn(len(slots), d)
        at = torch.tensor(slots, device="cuda", dtype=torch.int32)
        xc = conv1d_silu_step(x, w, bias, windows, at)
        dt, b, c = proj(xc)
        y = selective_state_step_slots(states, xc, dt, aneg, b, c, at)
        for r, slot in enumerate(slots):
            if slot >= 0:
                seen[slot].append(x[r:r + 1])
                outs[slot].append(y[r:r + 1])
            else:
                assert not y[r].any()

    def finish(slot):
        assert_close(f"slot {slot}", torch.cat(outs.pop(slot)), alone(torch.cat(seen.pop(slot))),
                     2e-5)

    prompts({4: 7, 0: 1, 2: 30})
    for _ in range(5):
        tokens([0, 2, -1, 4])
    finish(2)
    prompts({2: 3, 5: 12})       # a new request takes the slot
    for _ in range(4):
        tokens([5, 4, 2, 0])
    for slot in (0, 2, 4, 5):
        finish(slot)
    assert torch.isnan(windows[[1, 3]]).all() and torch.isnan(states[[1, 3]]).all()
    logits = F.linear(torch.randn(4, d, generator=g, device="cuda"), randn(100, d))
    assert sample_tokens(logits, torch.rand(4, device="cuda"), top_k=10).shape == (4,)


def test_prefill_of_an_end_past_the_tokens():
    """Lengths that the documentation does not allow: no access past the tokens."""
    model = _model()
    idx, _, _ = _prompts([6])
    with torch.no_grad():
        out = model.prefill(idx, torch.tensor([0, 4, 99], device="cuda"), {})
        want = model.prefill(idx, torch.tensor([0, 4, 6], device="cuda"), {})
    assert torch.equal(out, want)
