"""The next token from a model's logits, on the HIP kernels."""
from __future__ import annotations

import torch

from . import _native_packed
from ._native import dispatch
from .packed import _hip


def _setting(what: str, name: str, v, rows: torch.Size, ints: bool):
    """(the rows' settings or None, the value that then holds)."""
    if isinstance(v, torch.Tensor):
        if v.shape != rows or (v.is_floating_point() is ints) or v.is_complex() \
                or v.dtype == torch.bool:
            raise ValueError(f"{what}: {name} must be a number or a tensor of "
                             f"{'integers' if ints else 'floats'} of shape {tuple(rows)}; got "
                             f"{v.dtype} {tuple(v.shape)}")
        if ints:
            v = v if v.dtype in (torch.int32, torch.int64) else v.to(torch.int64)
        else:
            v = v.detach().to(torch.float32)
        return v.reshape(-1).contiguous(), 0
    return None, (int(v) if ints else float(v))


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=0,
                  top_p=1.0, min_p=0.0, return_logprobs: bool = False):
    """One token for each row of logits (..., V) (float32, bfloat16, float16), int64 (...).

    uniform (...) holds a number in [0, 1) per row, as torch.rand gives; the same numbers
    give the same tokens. Each setting is a number or a tensor of one per row (taken in
    float32), and 0 < temperature < inf scales the logits; then are kept, of the words by
    falling logit (the lower index first among equals), the top_k first (all if top_k < 1); of
    these those before which less than top_p of their probability lies (the first always; all
    from 1 on); and of these those with at least min_p times the likeliest one's
    probability. The token is the first kept word by index at which the running sum of the kept
    probabilities exceeds uniform times their total. Temperature 0: the largest logit, at its lowest
    index. NaN logits count as -inf. A row that has no logit above -inf, or settings that do not
    hold (temperature below 0 or infinite, min_p above 1, NaN), gives token -1.

    Fewer than 2^16 rows (of logits' leading dimensions), vocab up to 2^24. While it runs, a
    call of more than 4096 words holds 8 KB a row; and where top_k is a tensor, or off (below 1 or
    from vocab on), 8 KB more for each row and 8192 words above 8192, which in 16 bits is half
    of what the logits take.

    With return_logprobs also the log-probabilities (...) float32 of the tokens in the
    distributions that they were drawn from (NaN for token -1). Weights are formed in 64
    bits: which word a number falls on does not change from run to run."""
    what = "sample_tokens"
    _hip(what, logits, uniform)
    if logits.dim() < 1 or logits.shape[-1] < 1 or uniform.shape != logits.shape[:-1] \
            or not uniform.is_floating_point():
        raise ValueError(f"{what}: logits must be (..., vocab) and uniform (...) floats; got "
                         f"{tuple(logits.shape)}, {uniform.dtype} {tuple(uniform.shape)}")
    if logits.dtype not in _native_packed.DTYPES:
        raise RuntimeError(f"{what}: logits must be float32, bfloat16 or float16; got "
                           f"{logits.dtype}")
    lead = logits.shape[:-1]
    temperature, t = _setting(what, "temperature", temperature, lead, False)
    top_k, k = _setting(what, "top_k", top_k, lead, True)
    top_p, p = _setting(what, "top_p", top_p, lead, False)
    min_p, m = _setting(what, "min_p", min_p, lead, False)
    z = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    if (z.shape[1] > 1 and z.stride(1) != 1) or (z.shape[0] > 1 and z.stride(0) < z.shape[1]):
        z = z.clone(memory_format=torch.contiguous_format)
    if uniform.dim() != 1 or uniform.dtype is not torch.float32 or not uniform.is_contiguous():
        uniform = uniform.to(torch.float32).reshape(-1).contiguous()
    args = (z.detach() if z.requires_grad else z,
            uniform.detach() if uniform.requires_grad else uniform, temperature, top_k, top_p,
            min_p, [t, p, m], k)
    if not torch.compiler.is_compiling():
        _native_packed._check_sample(*args)
    tokens, logps = dispatch("sample")(*args)
    if len(lead) != 1:
        tokens, logps = tokens.view(lead), logps.view(lead)
    return (tokens, logps) if return_logprobs else tokens
