"""Sampling on the GPU against a word-by-word draw in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import packed_reference as ref
from mamba_metal_scan_amd import sample_tokens

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = math.inf


def check(z, u, **settings):
    """Tokens equal, log-probabilities within their fp32 rounding (and 2^-45 a word)."""
    rows = z.shape[0]
    tokens, logps = sample_tokens(
        z.cuda(), u.cuda(), return_logprobs=True,
        **{k: v.cuda() if torch.is_tensor(v) else v for k, v in settings.items()})
    assert tokens.dtype == torch.int64 and logps.dtype == F32
    for r in range(rows):
        own = {}
        for name, v in settings.items():
            v = v[r] if torch.is_tensor(v) else v
            own[name] = int(v) if name == "top_k" else float(torch.as_tensor(v, dtype=F32))
        token, logp = ref.sample(z[r].double(), float(u[r]), **own)
        assert int(tokens[r]) == token, (r, own, float(u[r]))
        if token < 0:
            assert math.isnan(float(logps[r]))
        else:
            assert abs(float(logps[r]) - logp) <= 2.0 ** -23 * abs(logp) + 1e-9, (r, own)


def _rand(rows, vocab, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(rows, vocab, generator=g)).to(dtype), torch.rand(rows, generator=g)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 1024, 5003])
def test_settings(vocab, dtype):
    z, u = _rand(6, vocab, dtype, vocab)
    for s in (dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=7), dict(top_k=vocab),
              dict(top_k=vocab + 9), dict(top_p=0.9), dict(top_p=0.3, temperature=1.7),
              dict(top_p=0.0), dict(top_p=-1.0), dict(min_p=0.05), dict(min_p=1.0),
              dict(top_k=20, top_p=0.8, min_p=0.01, temperature=0.9), dict(temperature=0.0),
              dict(temperature=0, top_k=3, top_p=0.5), dict(temperature=1e-30),
              dict(temperature=1e30, top_k=5)):
        check(z, u, **s)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_settings_of_the_rows(dtype):
    rows, vocab = 24, 2100
    z, u = _rand(rows, vocab, dtype, 5)
    g = torch.Generator().manual_seed(6)
    pick = lambda v: torch.tensor(v)[torch.randint(0, len(v), (rows,), generator=g)]   # noqa: E731
    check(z, u, temperature=pick([0.0, 0.5, 1.0, 1.5]), top_k=pick([0, -3, 1, 40, 3000]),
          top_p=pick([0.1, 0.9, 0.99, 1.0]), min_p=pick([0.0, 0.1]))
    check(z, u, top_k=pick([0, 3, 50]).to(torch.int32), top_p=pick([0.5, 0.9]).double())


def test_ties():
    """Words of one logit go by their index, at every border."""
    u = torch.tensor([0.0, 0.1, 0.25, 0.3, 0.5, 0.74999, 0.75, 0.99999994])
    flat = torch.zeros(8, 300)
    few = torch.tensor([1.0, 0.0, 1.0, -0.0, 1.0, -5.0, 0.0, 1.0]).repeat(8, 40)
    for dtype in (F32, BF16, F16):
        for z in (flat.to(dtype), few.to(dtype)):
            for s in (dict(), dict(top_k=3), dict(top_k=170), dict(top_p=0.5), dict(top_p=0.25),
                      dict(top_k=200, top_p=0.7), dict(top_p=0.01), dict(min_p=0.5),
                      dict(temperature=0.0)):
                check(z, u, **s)


def test_masks_infinities_and_nan():
    z, u = _rand(10, 400, F32, 9)
    z[0] = -INF                                  # a mask that leaves nothing
    z[1] = torch.finfo(F32).min                  # of the lowest value: all alike
    z[2, :399] = -INF
    z[3, ::2] = math.nan
    z[4] = math.nan
    z[5, [7, 300]] = INF
    z[6, 5] = INF
    z[7] = torch.finfo(F32).max
    z[8, 50:] = torch.finfo(F32).min
    z[9, 100:] = -INF
    for s in (dict(), dict(top_k=390), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.1),
              dict(temperature=0.0), dict(top_k=30, top_p=0.9, min_p=0.01)):
        check(z, u, **s)


def test_settings_that_do_not_hold():
    z, u = _rand(6, 100, F32, 2)
    check(z, u, temperature=torch.tensor([-1.0, math.nan, INF, 1.0, 1.0, 1.0]),
          min_p=torch.tensor([0.0, 0.0, 0.0, 1.5, math.nan, 0.0]),
          top_p=torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, math.nan]))


def test_uniform_numbers_outside():
    """Below 0 and NaN draw as 0 does, 1 and more the last word."""
    z, _ = _rand(4, 500, F32, 3)
    lo = sample_tokens(z.cuda(), torch.zeros(4, device="cuda"))
    hi = sample_tokens(z.cuda(), torch.full((4,), 2.0, device="cuda"))
    assert torch.equal(sample_tokens(z.cuda(), torch.full((4,), -1.0, device="cuda")), lo)
    assert torch.equal(sample_tokens(z.cuda(), torch.full((4,), math.nan, device="cuda")), lo)
    assert (lo == 0).all() and (hi == 499).all()


def test_shapes_and_layouts():
    z, _ = _rand(12, 700, BF16, 4)
    z, u = z.cuda(), torch.rand(12, device="cuda", dtype=torch.float64)
    want = sample_tokens(z, u, top_k=30)
    got = sample_tokens(z.view(3, 4, 700), u.view(3, 4), top_k=30)
    assert got.shape == (3, 4) and torch.equal(got.view(-1), want)
    wide = torch.randn(12, 900, device="cuda").to(BF16)
    wide[:, 100:800] = z
    assert torch.equal(sample_tokens(wide[:, 100:800], u, top_k=30), want)
    wide[:, 101:801] = z.clone()
    assert torch.equal(sample_tokens(wide[:, 101:801], u, top_k=30), want)   # odd addresses
    assert torch.equal(sample_tokens(z.t().contiguous().t(), u, top_k=30), want)
    assert sample_tokens(z[:0], u[:0]).shape == (0,)
    assert sample_tokens(z[0], u[0]).shape == ()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_vocabulary(dtype):
    z, u = _rand(3, 131072, dtype, 7)
    for s in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(min_p=0.02, top_k=1000)):
        check(z, u, **s)
    z, u = _rand(1, 300001, dtype, 8)
    check(z, u, top_p=0.9)


def test_frequencies():
    """20000 numbers spread evenly over [0, 1): each word is drawn in its share, within two."""
    n = 20000
    z = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.1])
    u = (torch.arange(n) + 0.5) / n
    t = sample_tokens(z.cuda().expand(n, 5), u.cuda(), temperature=0.8).cpu()
    p = torch.softmax(z.double() / 0.8, 0)
    assert (torch.bincount(t, minlength=5) - p * n).abs().max() <= 2


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_words_alike(dtype):
    """More words of one weight, or about it, than any list holds; k above 1024; a flat
    distribution; NaN among the words of a large k."""
    flat = torch.zeros(4, 20000)
    near, u = _rand(4, 40000, F32, 11, scale=0.05)
    masked = near.clone()
    masked[:, ::3] = math.nan
    masked[:, 1::3] = -INF
    steps = torch.randint(0, 3, (4, 30000), generator=torch.Generator().manual_seed(1)).float()
    for z in (flat, near, masked, steps):
        z = z.to(dtype)
        for s in (dict(top_p=0.5), dict(top_k=5000), dict(top_k=15000, top_p=0.7), dict(min_p=0.5),
                  dict(top_p=0.9, min_p=0.3), dict(top_k=1000), dict(top_k=39000), dict()):
            check(z, u, **s)


def test_middle_vocabularies():
    """About 8192 words (one part) and 1024 (one list), settings by row."""
    for vocab in (1023, 1025, 8191, 8192, 8193, 16385):
        z, u = _rand(8, vocab, F16, vocab)
        k = torch.tensor([0, 0, 0, 5, 900, 1500, 0, vocab])
        check(z, u, top_k=k, top_p=torch.tensor([1.0, 0.9, 0.2, 0.9, 0.9, 0.8, 1.0, 0.99]),
              min_p=torch.tensor([0.0, 0.0, 0.1, 0.0, 0.0, 0.0, 0.01, 0.0]))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_words_past_the_threads_maxima(dtype):
    """More than 16 vectors a thread; rows that start at any element; k at the bound's limits."""
    z, u = _rand(3, 140003, dtype, 21)
    for s in (dict(top_k=50, top_p=0.9), dict(top_k=2048, temperature=0.7),
              dict(top_k=2049, top_p=0.9), dict(top_p=0.9, min_p=0.001), dict(temperature=0.0)):
        check(z[:, 1:], u, **s)
    check(z[:1, 3:70000], u[:1], top_k=1000, top_p=0.95)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_words_in_order_and_few_words_left(dtype):
    """The likeliest words next to each other; masks that leave 1 and 30 words; one level."""
    up = torch.linspace(-8, 8, 20011).to(dtype)
    left = torch.full((20011,), -INF, dtype=dtype)
    left[7::667] = torch.randn(30, generator=torch.Generator().manual_seed(2)).to(dtype)
    one = torch.full((20011,), torch.finfo(dtype).min, dtype=dtype)
    one[20010] = 1.0
    low = torch.full((20011,), torch.finfo(dtype).min, dtype=dtype)
    z = torch.stack([up, up.flip(0), left, one, low])
    u = torch.tensor([0.1, 0.4, 0.9, 0.5, 0.77])
    for s in (dict(top_k=50), dict(top_k=1000, top_p=0.9), dict(top_k=20), dict(top_p=0.9), dict(),
              dict(min_p=0.02), dict(top_p=0.5, min_p=0.7), dict(temperature=0.0)):
        check(z, u, **s)


@pytest.mark.parametrize("vocab", [4097, 20000])
def test_top_p_and_min_p_at_the_bins(vocab):
    """min-p within, at the end of, before and behind the bin of top-p's border, by row."""
    z, u = _rand(12, vocab, F32, vocab)
    low = torch.tensor([0.5, 0.25, 0.3, 2.0 ** -0.0625, 0.001, 1e-9, 1e-30, 0.9, 1.0, 0.01, 0.07,
                        0.0])
    for p in (0.05, 0.5, 0.95, 0.9999):
        check(z, u, top_p=p, min_p=low, temperature=0.9)
    spread = (z * 0.02).clone()   # thousands of words a bin
    check(spread, u, top_p=0.6, min_p=low)


def test_a_very_large_vocabulary():
    """More than 256 parts: the draw goes through the row."""
    z, u = _rand(1, 2 ** 21 + 8195, F16, 3)
    check(z, u, top_p=0.8)
