"""Packed sequences and sampling, as cases to be measured.

Five operators that follow a prompt to its next token:

  conv1d_silu_packed           the short causal convolution with SiLU over the
                               tokens of several sequences behind each other,
                               with its gradients (packed documents) or from
                               and to windows of inputs (prompts)
  selective_scan_packed        the selective scan over the same, with its
                               gradients, or from and to states
  conv1d_silu_step             one token per row against a pool of windows,
  selective_state_step_slots   and of states, each row at its slot of the pool
  sample_tokens                temperature, top-k, top-p and min-p, and the
                               draw from a given uniform number, with the
                               drawn word's log-probability

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


def listed():
    return [
        # A batch of packed documents in training: as many tokens and channels
        # as the benchmark's scan (16 x 512 x 1536), x the left half of in_proj's output.
        dict(name="conv_train_bf16", kind="conv", tokens=8192, seqs=24, longest=2048, pad=0,
             dim=1536, taps=4, dtype="bf16", grad=True, carried=False),
        # Seven prompts of unlike length that continue from windows; an odd width.
        dict(name="conv_prompts_f32", kind="conv", tokens=1001, seqs=7, longest=509, pad=23,
             dim=1147, taps=4, dtype="f32", grad=False, carried=True),
        # The same batch of packed documents through the scan, in fp32.
        dict(name="scan_train_f32", kind="scan", tokens=8192, seqs=24, longest=2048, pad=0,
             dim=1536, states=16, dtype="f32", grad=True, carried=False),
        # Long documents in bf16: the most work.
        dict(name="scan_long_bf16", kind="scan", tokens=32768, seqs=9, longest=8192, pad=0,
             dim=2048, states=16, dtype="bf16", grad=True, carried=False),
        # Prompts of a wide model, some the next part of a long one, from and to states.
        dict(name="scan_prompts_bf16", kind="scan", tokens=4096, seqs=12, longest=2048, pad=128,
             dim=4096, states=16, dtype="bf16", grad=False, carried=True),
        # One prompt of 509 tokens: few channels, one sequence.
        dict(name="scan_prompt_f32", kind="scan", tokens=509, seqs=1, longest=509, pad=0,
             dim=640, states=16, dtype="f32", grad=False, carried=True),
        # The next token of four requests among 16 slots: launches and host time ...
        dict(name="conv_step_f32", kind="conv_step", rows=4, slots=16, dim=1536, taps=4,
             dtype="f32"),
        # ... and of 256 among 384, some rows being padding.
        dict(name="conv_step_bf16", kind="conv_step", rows=256, slots=384, dim=4096, taps=4,
             dtype="bf16"),
        dict(name="state_step_f32", kind="state_step", rows=4, slots=16, dim=1536, states=16,
             dtype="f32"),
        dict(name="state_step_bf16", kind="state_step", rows=256, slots=384, dim=4096, states=16,
             dtype="bf16"),
        # The draw for four requests of the benchmark's vocabulary ...
        dict(name="sample_f32", kind="sample", rows=4, vocab=32768, dtype="f32", mixed=False),
        # ... and for 256 with settings of their own, a large vocabulary.
        dict(name="sample_mixed_bf16", kind="sample", rows=256, vocab=131072, dtype="bf16",
             mixed=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    dim = _log(rng, lo, hi)
    return max(lo, dim // 64 * 64) if rng.random() < 0.7 else dim


def draw(rng):
    kind = rng.choice(["conv", "conv", "scan", "scan", "scan", "conv_step", "state_step",
                       "sample", "sample"])
    c = dict(kind=kind, dtype=rng.choice(["f32", "bf16", "bf16", "f16"]))
    if kind in ("conv", "scan"):
        c["dim"] = _width(rng, 16, 4096)
        if kind == "conv":
            c["taps"] = rng.choice([2, 3, 4, 4, 4, 8])
            most = (1 << 26) // c["dim"]
        else:
            c["states"] = rng.choice([1, 4, 8, 16, 16, 16, 16, 24, 32, 64])
            most = (1 << 30) // (c["dim"] * c["states"])
        c["tokens"] = max(1, min(_log(rng, 1, 32768), most))
        c["longest"] = max(-(-c["tokens"] // 8), min(c["tokens"], _log(rng, 1, 8192)))
        least = -(-c["tokens"] // c["longest"])
        c["seqs"] = min(512, max(_log(rng, 1, 128), least + least // 2))
        c["pad"] = rng.choice([0, 0, 1, 37])     # rows behind the last sequence
        c["grad"] = rng.random() < 0.6
        c["carried"] = rng.random() < 0.5        # from and to windows or states
    elif kind == "sample":
        c["vocab"] = _log(rng, 100, 131072)
        c["rows"] = max(1, min(_log(rng, 1, 512), (1 << 25) // c["vocab"]))
        c["mixed"] = rng.random() < 0.7
    else:
        c["dim"] = _width(rng, 16, 4096)
        c["taps" if kind == "conv_step" else "states"] = (
            rng.choice([2, 3, 4, 4, 8]) if kind == "conv_step"
            else rng.choice([1, 4, 8, 16, 16, 16, 32, 64]))
        c["rows"] = max(1, min(_log(rng, 1, 512), (1 << 25) // (c["dim"] * c.get("states", 4))))
        c["slots"] = c["rows"] + rng.choice([0, 1, 12, c["rows"]])
    return c


# ------------------------------------------------------------------- inputs

def _lengths(c, g):
    """Lengths of the case's sequences: unlike ones, some of no token and of one, that add up to
    its tokens, none longer than its longest."""
    n, total, top = c["seqs"], c["tokens"], c["longest"]
    if n == 1:
        return [total]
    w = torch.randn(n, generator=g, device=DEV).exp().double().cpu()
    w = (w / w.sum() * total).floor().clamp_(max=top).long().tolist()
    if n > 4:      # a sequence of no token and one of a single one
        w[1], w[2] = 0, 1
    left, i = total - sum(w), 0
    while left != 0:
        if n <= 4 or i % n not in (1, 2) or (i >= n and left > 0):
            step = min(left, top - w[i % n]) if left > 0 else max(left, -w[i % n])
            w[i % n] += step
            left -= step
        i += 1
    return w


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    s = {"case": c}
    if c["kind"] == "sample":
        rows, vocab = c["rows"], c["vocab"]
        z = 2.5 * randn(rows, vocab)
        z += 6.0 * (rand(rows, vocab) < 4.0 / vocab)    # a few words that the model likes
        z[:, vocab // 2] = -math.inf                    # a word that is not allowed
        s["logits"] = z.to(dtype)
        s["uniform"] = rand(rows)
        if c["mixed"]:
            pick = torch.randint(0, 4, (4, rows), generator=g, device=DEV)
            s["temperature"] = torch.tensor([0.6, 0.8, 1.0, 1.3], device=DEV)[pick[0]]
            s["top_k"] = torch.tensor([0, 20, 50, 1000], device=DEV)[pick[1]]
            s["top_p"] = torch.tensor([0.8, 0.9, 0.95, 1.0], device=DEV)[pick[2]]
            s["min_p"] = torch.tensor([0.0, 0.0, 0.02, 0.1], device=DEV)[pick[3]]
        else:
            s.update(temperature=0.8, top_k=50, top_p=0.9, min_p=0.0)
        return s
    d = c["dim"]
    if c["kind"] in ("conv", "scan"):
        lens = _lengths(c, g)
        rows = c["tokens"] + c["pad"]
        s["cu_seqlens"] = torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)
        s["lens"] = lens
    else:
        rows, pool = c["rows"], c["slots"]
        slots = torch.randperm(pool, generator=g, device=DEV)[:rows]
        if rows > 8:    # rows of a padded batch
            slots = torch.where(rand(rows) < 0.05, -1, slots)
        s["slots"] = slots.to(torch.int32)
    if c["kind"].startswith("conv"):
        k = c["taps"]
        s["x"] = randn(rows, 2 * d).to(dtype)[:, :d]    # the left half of in_proj's output
        s["weight"] = ((2.0 * rand(d, 1, k) - 1.0) / math.sqrt(k)).to(dtype)
        s["bias"] = ((2.0 * rand(d) - 1.0) / math.sqrt(k)).to(dtype)
        names = ["x", "weight", "bias"]
        if c["kind"] == "conv_step":
            s["window"] = randn(c["slots"], d, k - 1).to(dtype)
        else:
            s["window"] = randn(len(lens), d, k - 1).to(dtype) if c["carried"] else None
            names += ["window"] if c["carried"] else []
    else:
        n = c["states"]
        s["x"] = randn(rows, d).to(dtype)
        # dt as the block's gate gives it, between 0.001 and 0.1
        s["dt"] = (0.001 + 0.099 * torch.sigmoid(randn(rows, d))).to(dtype)
        a = torch.arange(1, n + 1, device=DEV) + 0.1 * randn(d, n)
        s["aneg"] = torch.nn.functional.softplus(a)
        s["B"] = randn(rows, n).to(dtype)
        s["C"] = randn(rows, n).to(dtype)
        names = ["x", "dt", "aneg", "B", "C"]
        if c["kind"] == "state_step":
            s["h"] = 0.3 * randn(c["slots"], d, n)
        else:
            s["h0"] = 0.3 * randn(len(lens), d, n) if c["carried"] else None
            names += ["h0"] if c["carried"] else []
    if c.get("grad"):
        s["leaves"] = names
        for name in names:
            s[name] = s[name].detach().requires_grad_(True)
        s["dy"] = randn(rows, d).to(dtype)
        if c["carried"]:
            s["dlast"] = (randn(len(lens), d, c["taps"] - 1).to(dtype) if c["kind"] == "conv"
                          else randn(len(lens), d, c["states"]))
    return s


# ------------------------------------------------- the package's operators

def _run_own(s):
    import mamba_metal_scan_amd as m
    c = s["case"]
    if c["kind"] == "sample":
        return list(m.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"],
                                    top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                    return_logprobs=True))
    if c["kind"] == "conv_step":
        return [m.conv1d_silu_step(s["x"], s["weight"], s["bias"], s["window"], s["slots"]),
                s["window"]]
    if c["kind"] == "state_step":
        return [m.selective_state_step_slots(s["h"], s["x"], s["dt"], s["aneg"], s["B"], s["C"],
                                             s["slots"]), s["h"]]
    if c["kind"] == "conv":
        out = m.conv1d_silu_packed(s["x"], s["weight"], s["bias"], s["cu_seqlens"],
                                   window=s["window"], return_window=c["carried"])
    else:
        out = m.selective_scan_packed(s["x"], s["dt"], s["aneg"], s["B"], s["C"],
                                      s["cu_seqlens"], h0=s["h0"], return_state=c["carried"])
    outs = list(out) if c["carried"] else [out]
    if not c["grad"]:
        return outs
    ups = [s["dy"], s["dlast"]] if c["carried"] else [s["dy"]]
    grads = torch.autograd.grad(outs, [s[name] for name in s["leaves"]], ups)
    return [o.detach() for o in outs] + list(grads)


# ------------------------------------------------------------- plain forms

def _padded(s):
    """Row numbers (seqs, longest) of the packed tokens, and which of them are tokens."""
    cu = s["cu_seqlens"].long()
    t = torch.arange(max(max(s["lens"]), 1), device=cu.device)
    at = cu[:-1, None] + t
    kept = at < cu[1:, None]
    return torch.where(kept, at, 0), kept


def _plain_conv(s):
    c = s["case"]
    k, d = c["taps"], c["dim"]
    x, dtype = s["x"].detach(), s["x"].dtype
    at, kept = _padded(s)
    w = s["weight"].detach().float().view(d, k)
    seqs, longest = at.shape
    xp = x.float()[at] * kept[..., None]
    before = (s["window"].detach().float().transpose(1, 2) if c["carried"]
              else xp.new_zeros(seqs, k - 1, d))
    full = torch.cat([before, xp], 1)                       # (seqs, k - 1 + longest, d)
    pre = s["bias"].detach().float().expand(seqs, longest, d).clone()
    for j in range(k):
        pre += w[:, j] * full[:, j:j + longest]
    sig = 1.0 / (1.0 + torch.exp(-pre))
    out = x.new_zeros(x.shape)
    out[at[kept]] = (pre * sig)[kept].to(dtype)
    outs = [out]
    if c["carried"]:
        n = torch.tensor(s["lens"], device=x.device)
        last = n[:, None] + torch.arange(k - 1, device=x.device)
        outs.append(full.gather(1, last[..., None].expand(-1, -1, d)).transpose(1, 2).to(dtype))
    if not c["grad"]:
        return outs
    ds = s["dy"].float()[at] * kept[..., None] * sig * (1.0 + pre * (1.0 - sig))
    dfull = torch.zeros_like(full)
    dw = torch.empty_like(w)
    for j in range(k):
        dfull[:, j:j + longest] += w[:, j] * ds
        dw[:, j] = (ds * full[:, j:j + longest]).sum((0, 1))
    if c["carried"]:
        dfull.scatter_add_(1, last[..., None].expand(-1, -1, d),
                           s["dlast"].float().transpose(1, 2))
    dx = x.new_zeros(x.shape)
    dx[at[kept]] = dfull[:, k - 1:][kept].to(dtype)
    outs += [dx, dw.view(d, 1, k).to(dtype), ds.sum((0, 1)).to(dtype)]
    if c["carried"]:
        outs.append(dfull[:, :k - 1].transpose(1, 2).to(dtype))
    return outs


def _plain_scan(s):
    c = s["case"]
    x, dtype = s["x"].detach(), s["x"].dtype
    at, kept = _padded(s)
    seqs, longest = at.shape
    m = kept[..., None].float()
    an = s["aneg"].detach().float()
    xs, dts = x.float()[at] * m, s["dt"].detach().float()[at] * m
    bs, cs = s["B"].detach().float()[at] * m, s["C"].detach().float()[at] * m
    h = (s["h0"].detach().clone() if c["carried"]
         else xs.new_zeros(seqs, c["dim"], c["states"]))
    first = h
    hs = []
    ys = torch.empty_like(xs)
    for t in range(longest):    # (padded steps keep the state: dt = 0 there)
        dt = dts[:, t, :, None]
        h = torch.exp(-dt * an) * h + dt * xs[:, t, :, None] * bs[:, t, None]
        ys[:, t] = (h * cs[:, t, None]).sum(-1)
        if c["grad"]:
            hs.append(h)
    y = x.new_zeros(x.shape)
    y[at[kept]] = ys[kept].to(dtype)
    outs = [y, h] if c["carried"] else [y]
    if not c["grad"]:
        return outs
    dys = s["dy"].float()[at] * m
    u = s["dlast"].clone() if c["carried"] else torch.zeros_like(h)
    dxs, ddts = torch.empty_like(xs), torch.empty_like(xs)
    dbs, dcs = torch.empty_like(bs), torch.empty_like(cs)
    da = torch.zeros_like(an)
    for t in range(longest - 1, -1, -1):
        dt = dts[:, t, :, None]
        gr = u + dys[:, t, :, None] * cs[:, t, None]
        u = torch.exp(-dt * an) * gr
        q = u * (hs[t - 1] if t else first)
        gb = (gr * bs[:, t, None]).sum(-1)
        dxs[:, t] = dts[:, t] * gb
        ddts[:, t] = xs[:, t] * gb - (an * q).sum(-1)
        dbs[:, t] = (gr * (dts[:, t] * xs[:, t])[..., None]).sum(1)
        dcs[:, t] = (dys[:, t, :, None] * hs[t]).sum(1)
        da -= (dt * q).sum(0)
    for like, v in ((s["x"], dxs), (s["dt"], ddts), (None, da), (s["B"], dbs), (s["C"], dcs)):
        if like is None:
            outs.append(v)
        else:
            full = torch.zeros_like(like.detach())
            full[at[kept]] = v[kept].to(dtype)
            outs.append(full)
    return outs + [u] if c["carried"] else outs


def _plain_conv_step(s):
    c = s["case"]
    x = s["x"]
    live = s["slots"] >= 0
    slots = s["slots"][live].long()
    win = torch.cat([s["window"][slots], x[live][..., None]], 2)
    w = s["weight"].float().view(c["dim"], c["taps"])
    pre = s["bias"].float() + (win.float() * w).sum(-1)
    out = x.new_zeros(x.shape)
    out[live] = (pre / (1.0 + torch.exp(-pre))).to(x.dtype)
    s["window"][slots] = win[..., 1:]
    return [out, s["window"]]


def _plain_state_step(s):
    x = s["x"]
    live = s["slots"] >= 0
    slots = s["slots"][live].long()
    dt = s["dt"][live].float()[..., None]
    h = (torch.exp(-dt * s["aneg"]) * s["h"][slots]
         + dt * x[live].float()[..., None] * s["B"][live].float()[:, None])
    y = x.new_zeros(x.shape)
    y[live] = (h * s["C"][live].float()[:, None]).sum(-1).to(x.dtype)
    s["h"][slots] = h
    return [y, s["h"]]


def _setting(v, rows, device):
    v = v if torch.is_tensor(v) else torch.full((rows,), v, device=device)
    return v.double()[:, None]


def _plain_sample(s):
    """In 64 bits: where the running sums cross a border decides the token."""
    z = s["logits"].double()
    rows, vocab = z.shape
    t, k, p, low = (_setting(s[name], rows, z.device)
                    for name in ("temperature", "top_k", "top_p", "min_p"))
    z, order = z.sort(dim=1, descending=True, stable=True)
    w = torch.exp((z - z[:, :1]) / t)
    rank = torch.arange(vocab, device=z.device)
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    run = w.cumsum(1)
    before = run - w
    w = torch.where((p >= 1.0) | (before < p * run[:, -1:]) | (rank == 0), w, 0.0)
    w = torch.where(w >= low, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    run = w.cumsum(1)
    above = run > s["uniform"].double()[:, None] * run[:, -1:]
    token = above.to(torch.uint8).argmax(1)
    share = w.gather(1, token[:, None]) / run[:, -1:]
    return [token, torch.log(share)[:, 0].float()]


def _run_plain(s):
    return {"conv": _plain_conv, "scan": _plain_scan, "conv_step": _plain_conv_step,
            "state_step": _plain_state_step, "sample": _plain_sample}[s["case"]["kind"]](s)


def run(s):
    return _run_own(s) if own else _run_plain(s)


# --------------------------------------------------------------------- work

def work(case):
    """Each input read and each output written once. Operations: the convolution's products, the
    scan's update and sum (an exponential counted as one), and their gradients."""
    c = case
    es = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "sample":
        return dict(bytes=es * c["rows"] * c["vocab"] + 16 * c["rows"],
                    flops=4 * c["rows"] * c["vocab"])
    d = c["dim"]
    if c["kind"] == "conv_step":
        r, k = c["rows"], c["taps"]
        return dict(bytes=es * (2 * r * d * (k - 1) + 2 * r * d + d * (k + 1)) + 4 * r,
                    flops=(2 * k + 5) * r * d)
    if c["kind"] == "state_step":
        r, n = c["rows"], c["states"]
        return dict(bytes=8 * r * d * n + es * r * (3 * d + 2 * n) + 4 * d * n + 4 * r,
                    flops=7 * r * d * n)
    rows, seqs = c["tokens"] + c["pad"], c["seqs"]
    if c["kind"] == "conv":
        k = c["taps"]
        ends = 2 * seqs * d * (k - 1) * es if c["carried"] else 0
        once = es * (2 * rows * d + d * (k + 1)) + ends
        back = es * (3 * rows * d + 2 * d * (k + 1)) + ends
        return dict(bytes=once + (back if c["grad"] else 0),
                    flops=((6 * k + 15) if c["grad"] else (2 * k + 5)) * c["tokens"] * d)
    n = c["states"]
    ends = 8 * seqs * d * n if c["carried"] else 0
    once = es * rows * (3 * d + 2 * n) + 4 * d * n + ends
    back = es * rows * (5 * d + 4 * n) + 8 * d * n + ends
    return dict(bytes=once + (back if c["grad"] else 0),
                flops=(27 if c["grad"] else 7) * c["tokens"] * d * n)


# ---------------------------------------------------- the same in 64 bits

def _each(s):
    i = 0
    for q, n in enumerate(s["lens"]):
        yield q, slice(i, i + n), n
        i += n


def _exact_conv(s):
    c = s["case"]
    k, d = c["taps"], c["dim"]
    leaves = {name: s[name].detach().double().requires_grad_(c["grad"])
              for name in ("x", "weight", "bias")}
    win = (s["window"].detach().double() if c["carried"]
           else torch.zeros(c["seqs"], d, k - 1, dtype=torch.float64, device=DEV))
    win.requires_grad_(c["grad"])
    outs, ends = [], []
    for q, part, n in _each(s):
        row = torch.cat([win[q], leaves["x"][part].t()], 1)           # (d, k - 1 + n)
        ends.append(row[:, n:])
        if n:
            pre = torch.nn.functional.conv1d(row[None], leaves["weight"], leaves["bias"],
                                             groups=d)[0]
            outs.append(torch.nn.functional.silu(pre).t())
    outs.append(torch.zeros(c["pad"], d, dtype=torch.float64, device=DEV))
    res = [torch.cat(outs)] + ([torch.stack(ends)] if c["carried"] else [])
    if not c["grad"]:
        return res
    wrt = list(leaves.values()) + ([win] if c["carried"] else [])
    ups = [s["dy"].double()] + ([s["dlast"].double()] if c["carried"] else [])
    return [r.detach() for r in res] + list(torch.autograd.grad(res, wrt, ups))


def _exact_scan(s):
    """Channel by channel block, all the tokens' states kept: h over a sequence as a doubling
    scan of the pairs (decay, input) along time, the adjoint the same backwards in time."""
    c = s["case"]
    total, n_st = c["tokens"] + c["pad"], c["states"]

    def doubling(a, b, h):
        # b_t <- h_t of h_t = a_t h_{t-1} + b_t, h_{-1} = h
        b = b.clone()
        b[0] += a[0] * h
        a, step = a.clone(), 1
        while step < len(a):
            b[step:] = b[step:] + a[step:] * b[:-step]
            a[step:] = a[step:] * a[:-step]
            step *= 2
        return b

    x, dt, bb, cc = (s[name].detach().double() for name in ("x", "dt", "B", "C"))
    an = s["aneg"].detach().double()
    y, grad = torch.zeros_like(x), c["grad"]
    h0 = s["h0"].detach().double() if c["carried"] else x.new_zeros(c["seqs"], c["dim"], n_st)
    hl = h0.clone()
    dx, ddt, db, dc = (torch.zeros_like(v) for v in (x, dt, bb, cc))
    da, dh0 = torch.zeros_like(an), torch.zeros_like(h0)
    dlast = s["dlast"].double() if grad and c["carried"] else torch.zeros_like(h0)
    for q, part, n in _each(s):
        dh0[q] = dlast[q]
        if n == 0:
            continue
        step = max(1, (1 << 26) // (n * n_st))
        for lo in range(0, c["dim"], step):
            ch = slice(lo, min(c["dim"], lo + step))
            xs, ds = x[part, ch, None], dt[part, ch, None]
            a = torch.exp(-ds * an[ch])
            h = doubling(a, ds * xs * bb[part, None], h0[q, ch])
            y[part, ch] = torch.einsum("tdn,tn->td", h, cc[part])
            hl[q, ch] = h[-1]
            if not grad:
                continue
            gy = s["dy"][part, ch].double()[..., None] * cc[part, None]
            # G_t = gy_t + a_{t+1} G_{t+1}, from the last
            ahead = torch.cat([a[1:], torch.ones_like(a[:1])])
            gr = doubling(ahead.flip(0), gy.flip(0), dlast[q, ch]).flip(0)
            prev = torch.cat([h0[q, ch][None], h[:-1]])
            da_t = gr * prev * a                       # gradient of log a
            gb = torch.einsum("tdn,tn->td", gr, bb[part])
            dx[part, ch] = gb * ds[..., 0]
            ddt[part, ch] = gb * xs[..., 0] - torch.einsum("tdn,dn->td", da_t, an[ch])
            da[ch] -= torch.einsum("tdn,td->dn", da_t, ds[..., 0])
            db[part] += torch.einsum("tdn,td->tn", gr, (ds * xs)[..., 0])
            dc[part] += torch.einsum("tdn,td->tn", h, s["dy"][part, ch].double())
            dh0[q, ch] = a[0] * gr[0]
    outs = [y, hl] if c["carried"] else [y]
    if grad:
        outs += [dx, ddt, da, db, dc] + ([dh0] if c["carried"] else [])
    assert len(y) == total
    return outs


def _exact_sample(s):
    """Row by row, from the words in their order: the first of them that each setting leaves, as
    a count."""
    def of(name, r):
        v = s[name]
        return float(v[r] if torch.is_tensor(v) else torch.tensor(v, dtype=torch.float32))

    tokens, logps = [], []
    for r, row in enumerate(s["logits"]):
        words = torch.argsort(row, descending=True, stable=True)
        w = torch.softmax(row[words].double() / of("temperature", r), 0)
        k, p = int(of("top_k", r)), of("top_p", r)
        n = min(k, len(w)) if k > 0 else len(w)
        if p < 1.0:     # the words before the first at which the sum reaches its share, and it
            run = w[:n].cumsum(0)
            n = min(n, int((run < p * run[-1]).sum()) + 1)
        n = min(n, max(1, int((w >= of("min_p", r) * w[0]).sum())))
        at, where = words[:n].sort()
        w = w[:n][where]
        run = w.cumsum(0)
        i = int(torch.searchsorted(run, s["uniform"][r].double() * run[-1], right=True))
        i = min(i, n - 1)
        tokens.append(at[i])
        logps.append(w[i].log() - run[-1].log())
    return [torch.stack(tokens), torch.stack(logps)]


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "conv":
        return _exact_conv(s)
    if c["kind"] == "scan":
        return _exact_scan(s)
    if c["kind"] == "sample":
        return _exact_sample(s)
    slots = s["slots"].tolist()
    live = [r for r, at in enumerate(slots) if at >= 0]
    to = [slots[r] for r in live]
    out = torch.zeros(s["x"].shape, dtype=torch.float64, device=DEV)
    if c["kind"] == "conv_step":
        pool = s["window"].double()
        win = torch.cat([pool[to], s["x"][live].double().unsqueeze(2)], 2)
        pre = torch.einsum("rdk,dk->rd", win, s["weight"].double()[:, 0]) + s["bias"].double()
        out[live] = torch.nn.functional.silu(pre)
        pool[to] = win[:, :, 1:]
        return [out, pool]
    pool = s["h"].double()
    dt, x = s["dt"][live].double(), s["x"][live].double()
    h = pool[to] * torch.exp(-dt.unsqueeze(2) * s["aneg"].double())
    h += torch.einsum("rd,rn->rdn", dt * x, s["B"][live].double())
    out[live] = torch.einsum("rdn,rn->rd", h, s["C"][live].double())
    pool[to] = h
    return [out, pool]
