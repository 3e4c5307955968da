"""Losses of a language model's head, as cases to be measured.

Three operators, each beside `cross_entropy` in the package:

  linear_cross_entropy   cross entropy of the logits hidden @ weight.T, the
                         logits never held whole; with both gradients
                         (training), or one loss per row (scoring text,
                         the last token of a batch of sequences)
  distill_loss           distillation of given logits from a teacher's top
                         logits: temperature^2 KL(softmax over the teacher's
                         k words || softmax over the student's vocabulary)
  linear_distill_loss    the same from the hidden states, without the logits

`listed()` gives the named cases, `draw(rng)` another case of the same
ranges, `prepare` what a program holds before the call, `run` the pass (in
elementary torch operations, or with `own` set the package's operators),
`work` the bytes and operations the pass cannot do without, `exact` the same
outputs in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORE = -100


def listed():
    return [
        # One training batch of the benchmark's 80M model (16 x 512 tokens,
        # width 640, 32768 words), in fp32 as the model trains by default ...
        dict(name="lce_train_f32", kind="lce", rows=8192, dim=640, vocab=32768, dtype="f32",
             reduction="mean", grad=True),
        # ... and in bf16, as under autocast.
        dict(name="lce_train_bf16", kind="lce", rows=8192, dim=640, vocab=32768, dtype="bf16",
             reduction="mean", grad=True),
        # The head of a wide model with a large vocabulary: the most work.
        dict(name="lce_wide_bf16", kind="lce", rows=8192, dim=4096, vocab=131072, dtype="bf16",
             reduction="mean", grad=True),
        # A ragged batch of the 18M model in fp16, an odd vocabulary, the
        # sum of the losses (gradient accumulation).
        dict(name="lce_ragged_f16", kind="lce", rows=1001, dim=384, vocab=50257, dtype="f16",
             reduction="sum", grad=True),
        # Scoring one prompt of 509 tokens (as the 18M model's, at a wider
        # width): a log-probability per token, no gradient.
        dict(name="lce_score_bf16", kind="lce", rows=509, dim=2048, vocab=50257, dtype="bf16",
             reduction="none", grad=False),
        # The next token of four sequences against the 80M model's head.
        dict(name="lce_token_f32", kind="lce", rows=4, dim=640, vocab=32768, dtype="f32",
             reduction="none", grad=False),
        # Distillation of the 80M model's logits from a teacher's 64 top words.
        dict(name="distill_train_f32", kind="distill", rows=8192, k=64, vocab=32768,
             dtype="f32", temperature=2.0, reduction="mean", grad=True),
        # bf16 logits over an odd vocabulary, rows not 16-byte aligned.
        dict(name="distill_odd_bf16", kind="distill", rows=4096, k=20, vocab=50257,
             dtype="bf16", temperature=1.0, reduction="mean", grad=True),
        # A few rows of a small vocabulary: launches and host time.
        dict(name="distill_small", kind="distill", rows=8, k=5, vocab=1001, dtype="f32",
             temperature=1.0, reduction="mean", grad=True),
        # Distillation of the same batch from the hidden states.
        dict(name="ldistill_train_bf16", kind="ldistill", rows=8192, dim=640, k=64, vocab=32768,
             dtype="bf16", temperature=2.0, reduction="mean", grad=True),
        # A wider student, a large vocabulary, fewer words kept.
        dict(name="ldistill_wide_bf16", kind="ldistill", rows=4096, dim=2048, k=32, vocab=131072,
             dtype="bf16", temperature=1.5, reduction="mean", grad=True),
        # A short fp32 batch of the 18M model.
        dict(name="ldistill_f32", kind="ldistill", rows=509, dim=384, k=16, vocab=32768,
             dtype="f32", temperature=2.0, reduction="mean", grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lce", "lce", "lce", "distill", "distill", "ldistill", "ldistill"])
    c = dict(kind=kind, dtype=rng.choice(["f32", "bf16", "bf16", "f16"]))
    vocab = _log(rng, 1000, 131072)
    if rng.random() < 0.5:
        vocab = max(1000, vocab // 128 * 128)   # padded vocabularies
    c["vocab"] = vocab
    if kind == "distill":
        c["rows"] = max(1, min(8192, _log(rng, 1 << 13, 1 << 28) // vocab))
    else:
        dim = _log(rng, 64, 4096)
        if rng.random() < 0.8:
            dim = max(64, dim // 64 * 64)       # widths of models, else any
        c["dim"] = dim
        # fp32 products cost about eight times bf16's
        most = (1 << 42) >> (3 if c["dtype"] == "f32" else 0)
        c["rows"] = max(1, min(_log(rng, 1, 8192), most // (dim * vocab)))
    if kind != "lce":
        c["k"] = rng.choice([1, 5, 8, 16, 20, 32, 50, 64, 100, 128])
        c["temperature"] = rng.choice([1.0, 1.0, 1.5, 2.0, 4.0])
    c["grad"] = rng.random() < 0.75
    # Training takes a mean, a sum or weighted rows, scoring the rows' losses.
    c["reduction"] = rng.choice(["mean", "mean", "sum", "none"]) if c["grad"] else "none"
    return c


# ------------------------------------------------------------------- inputs

def _top_words(z, k, g):
    """The k top logits (and their words) of a teacher whose logits are the
    student's z with noise of their own; a few rows keep fewer than k words
    (padded with word -1), as a teacher cut at a probability sends them."""
    t = z.float() + torch.randn(z.shape, generator=g, device=z.device)
    values, ids = t.topk(k, dim=1)
    short = torch.rand(len(z), 1, generator=g, device=z.device) < 0.1
    at = torch.arange(k, device=z.device)
    ids = torch.where(short & (at >= (k + 1) // 2), -1, ids)
    return values, ids


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = DTYPES[c["dtype"]]
    rows, vocab = c["rows"], c["vocab"]
    s = {"case": c}
    if c["grad"]:   # the loss's gradient, from what later code makes of it
        shape = (rows,) if c["reduction"] == "none" else ()
        s["upstream"] = 0.5 + torch.rand(shape, generator=g, device=DEV)
    targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    if c["kind"] == "distill":
        z = 2.5 * torch.randn(rows, vocab, generator=g, device=DEV)
        s["logits"] = z.to(dtype).requires_grad_(c["grad"])
        parts = [_top_words(z[i:i + 1024], c["k"], g) for i in range(0, rows, 1024)]
    else:
        dim = c["dim"]
        # A head at the model's initial scale; hidden states of unit scale
        # that lean to their target's row by between nothing and enough for a
        # logit of 10 (a word that the model is sure of).
        w = 0.02 * torch.randn(vocab, dim, generator=g, device=DEV)
        lean = 10.0 / (0.02 * 0.02 * dim) * torch.rand(rows, 1, generator=g, device=DEV)
        h = torch.randn(rows, dim, generator=g, device=DEV) + lean * w[targets]
        s["hidden"] = h.to(dtype).requires_grad_(c["grad"])
        s["weight"] = w.to(dtype).requires_grad_(c["grad"])
        if c["kind"] == "lce":
            pad = torch.rand(rows, generator=g, device=DEV) < 0.1   # padding, ignored
            pad[0] = False
            s["targets"] = torch.where(pad, IGNORE, targets)
            return s
        hb, wb = h.to(torch.bfloat16), w.to(torch.bfloat16)
        parts = [_top_words(hb[i:i + 1024] @ wb.t(), c["k"], g) for i in range(0, rows, 1024)]
    s["teacher_logits"] = torch.cat([p[0] for p in parts])
    s["teacher_ids"] = torch.cat([p[1] for p in parts])
    return s


# ------------------------------------------------- the package's operators

def _run_own(s):
    from mamba_metal_scan_amd import distill_loss, linear_cross_entropy, linear_distill_loss
    c = s["case"]
    if c["kind"] == "distill":
        leaves = [s["logits"]]
        loss = distill_loss(*leaves, s["teacher_logits"], s["teacher_ids"],
                            temperature=c["temperature"], reduction=c["reduction"])
    else:
        leaves = [s["hidden"], s["weight"]]
        if c["kind"] == "lce":
            loss = linear_cross_entropy(*leaves, s["targets"], ignore_index=IGNORE,
                                        reduction=c["reduction"])
        else:
            loss = linear_distill_loss(*leaves, s["teacher_logits"], s["teacher_ids"],
                                       temperature=c["temperature"],
                                       reduction=c["reduction"])
    if not c["grad"]:
        return [loss]
    return [loss.detach(), *torch.autograd.grad(loss, leaves, s["upstream"])]


# ------------------------------------------------------------- plain forms

def _softmax_parts(y):
    """exp(y - max), its row sums, and the log-sum-exp of the rows of y."""
    m = y.amax(dim=1, keepdim=True)
    e = torch.exp(y - m)
    total = e.sum(dim=1, keepdim=True)
    return e, total, (m + torch.log(total)).squeeze(1)


def _reduced(losses, counted, s):
    """The loss from the rows' losses, and the gradient of each row's."""
    c = s["case"]
    count = counted.sum()
    loss = losses
    if c["reduction"] != "none":
        loss = losses.double().sum()
        loss = (loss / count if c["reduction"] == "mean" else loss).float()
    if not c["grad"]:
        return loss, None
    scale = s["upstream"] / count if c["reduction"] == "mean" else s["upstream"]
    return loss, torch.where(counted, scale, 0.0).unsqueeze(1)


def _plain_cross_entropy(s):
    c = s["case"]
    hidden, weight = s["hidden"].detach(), s["weight"].detach()
    h, w, t = hidden.float(), weight.float(), s["targets"]
    kept = t != IGNORE
    at = torch.where(kept, t, 0).unsqueeze(1)
    z = h @ w.t()
    e, total, lse = _softmax_parts(z)
    losses = torch.where(kept, lse - z.gather(1, at).squeeze(1), 0.0)
    loss, scale = _reduced(losses, kept, s)
    if not c["grad"]:
        return [loss]
    dz = e / total
    dz.scatter_add_(1, at, torch.full_like(scale, -1.0))
    dz *= scale
    return [loss, (dz @ w).to(hidden.dtype), (dz.t() @ h).to(weight.dtype)]


def _teacher(values, ids, temperature):
    """The teacher's probabilities over its kept words (0 on padding)."""
    y = torch.where(ids >= 0, values.float() / temperature, -math.inf)
    e = torch.exp(y - y.amax(dim=1, keepdim=True))
    return e / e.sum(dim=1, keepdim=True)


def _plain_distill(z, s):
    """The loss and its gradient to the fp32 logits z."""
    c = s["case"]
    temperature = c["temperature"]
    ids = s["teacher_ids"]
    q = _teacher(s["teacher_logits"], ids, temperature)
    at = ids.clamp(min=0)
    y = z / temperature
    e, total, lse = _softmax_parts(y)
    terms = torch.where(q > 0, q * (torch.log(q) - y.gather(1, at) + lse.unsqueeze(1)), 0.0)
    losses = temperature * temperature * terms.sum(dim=1)
    loss, scale = _reduced(losses, (q > 0).any(dim=1), s)
    if not c["grad"]:
        return loss, None
    dz = e / total
    dz.scatter_add_(1, at, -q)
    dz *= temperature * scale
    return loss, dz


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "lce":
        return _plain_cross_entropy(s)
    if c["kind"] == "distill":
        logits = s["logits"].detach()
        loss, dz = _plain_distill(logits.float(), s)
        return [loss, dz.to(logits.dtype)] if c["grad"] else [loss]
    hidden, weight = s["hidden"].detach(), s["weight"].detach()
    h, w = hidden.float(), weight.float()
    loss, dz = _plain_distill(h @ w.t(), s)
    if not c["grad"]:
        return [loss]
    return [loss, (dz @ w).to(hidden.dtype), (dz.t() @ h).to(weight.dtype)]


def run(s):
    return _run_own(s) if own else _run_plain(s)


# --------------------------------------------------------------------- work

def work(case):
    """Each input read and each output written once; of the products the
    logits once and the two gradients, 2 rows dim vocab operations each."""
    c = case
    es = 4 if c["dtype"] == "f32" else 2
    rows, vocab = c["rows"], c["vocab"]
    passes = 2 if c["grad"] else 1
    top = 0 if c["kind"] == "lce" else rows * c["k"] * (4 + 8)
    if c["kind"] == "distill":
        return dict(bytes=passes * es * rows * vocab + top, flops=4 * passes * rows * vocab)
    dim = c["dim"]
    ends = rows * (8 + 4) if c["kind"] == "lce" else top
    return dict(bytes=passes * es * (rows + vocab) * dim + ends,
                flops=(6 if c["grad"] else 2) * rows * dim * vocab)


# ---------------------------------------------------- the same in 64 bits

def _exact_rows(z, c, s, rows):
    """The losses of the logits z of the given rows, and their gradients to z
    with a loss's gradient of 1 each."""
    logp_of = torch.log_softmax
    if c["kind"] == "lce":
        t = s["targets"][rows]
        logp = logp_of(z, dim=1)
        idx = torch.arange(len(t), device=z.device)
        ignored = t == IGNORE
        word = t.masked_fill(ignored, 0)
        loss = -logp[idx, word]
        dz = logp.exp_()
        dz[idx, word] -= 1.0
        loss[ignored] = 0.0
        dz[ignored] = 0.0
        return loss, dz
    tau = c["temperature"]
    ids = s["teacher_ids"][rows]
    t = s["teacher_logits"][rows].double()
    logq = logp_of((t / tau).masked_fill(ids < 0, -math.inf), dim=1)
    logp = logp_of(z / tau, dim=1)
    q = logq.exp()
    word = ids.clamp_min(0)
    diff = (logq - logp.gather(1, word)).masked_fill(ids < 0, 0.0)
    loss = tau * tau * (q * diff).sum(1)
    return loss, tau * logp.exp_().scatter_add_(1, word, -q)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    n = c["rows"]
    share = 1.0
    if c["reduction"] == "mean":   # (every row keeps words of the teacher)
        share = (s["targets"] != IGNORE).sum().double() if c["kind"] == "lce" else float(n)
    h = s["hidden"].detach().double() if "hidden" in s else None
    w = s["weight"].detach().double() if "weight" in s else None
    losses, dlogits, dhidden = [], [], []
    dweight = torch.zeros_like(w) if w is not None and c["grad"] else None
    step = max(1, (1 << 27) // c["vocab"])
    for i in range(0, n, step):
        part = slice(i, min(n, i + step))
        z = s["logits"].detach()[part].double() if h is None else h[part] @ w.t()
        loss, dz = _exact_rows(z, c, s, part)
        losses.append(loss)
        if not c["grad"]:
            continue
        up = s["upstream"].double()
        dz *= (up[part].unsqueeze(1) if up.dim() else up) / share
        if h is None:
            dlogits.append(dz)
        else:
            dhidden.append(dz @ w)
            dweight += dz.t() @ h[part]
    loss = torch.cat(losses)
    if c["reduction"] != "none":
        loss = loss.sum() / share
    if not c["grad"]:
        return [loss]
    if h is None:
        return [loss, torch.cat(dlogits)]
    return [loss, torch.cat(dhidden), dweight]
