"""The block's conv and scan over packed sequences, and one token by slot.

Prompts and documents are of unlike lengths. ``conv1d_silu`` and ``selective_scan``
take rectangular batches that start from nothing; these take sequences that lie
behind each other in the rows of (L, ...) tensors, ``cu_seqlens`` (S + 1 integers
on the device) naming each one's first row and the end of the last, with no
padding between them:

* ``conv1d_silu_packed`` and ``selective_scan_packed``: no input of one sequence
  reaches another. Each may start from what came before it (``window``, the last
  K - 1 inputs of the conv; ``h0``, the scan's states) and gives what the next part
  needs. Differentiable in all of these, once.
* ``conv1d_silu_step`` and ``selective_state_step_slots``: one token per row, row r
  against entry ``slots[r]`` of a pool of windows or states, updated in place. For
  serving requests that come and go (no gradients).

Activations are float32, bfloat16 or float16, states float32. The lengths stay on the
device: no call waits for the GPU, and a captured call replays with other lengths in
``cu_seqlens`` (or other ``slots``).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native, _native_packed
from ._native import HipScanError, dispatch


def _hip(what: str, *ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            break
    else:
        if torch.version.hip is not None:
            return
    raise RuntimeError(f"{what} needs its tensors on the ROCm device; got "
                       + ", ".join(str(t.device) for t in ts if t is not None))


def _records(*ts: Optional[torch.Tensor]) -> bool:
    """Whether autograd records what becomes of ts (requires_grad, or a forward-mode tangent):
    else the forward runs without it."""
    if torch.compiler.is_compiling():
        return True
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    # (tangents there are only within a dual level)
    return (getattr(forward_ad, "_current_level", 0) >= 0
            and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The 2-D t, or a copy of it whose rows the kernels read."""
    if t.dim() != 2 or _native_packed.rows_ok(t):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t, contiguous and 16-byte aligned."""
    if t is None:
        return None
    t = t.contiguous()
    # (the address is known only outside tracing: the op checks it)
    return t if torch.compiler.is_compiling() or t.data_ptr() % 16 == 0 else t.clone()


def _once(what: str) -> None:
    if torch.is_grad_enabled() and not torch.compiler.is_compiling():
        raise HipScanError(f"{what} is once differentiable (create_graph is not supported)")


class SelectiveScanPackedHIP(torch.autograd.Function):
    """selective_scan_packed on the HIP kernels: (y, h_last) or y."""

    @staticmethod
    def run(x, dt, aneg, b_in, c_in, cu, h0, return_state, with_ckpt):
        """((y, h_last, ckpt), the operands as the kernels read them)."""
        ts = (x, dt, aneg, b_in, c_in, cu, h0)
        # (while tracing the registered op checks itself)
        if torch.compiler.is_compiling() or not _native_packed._scan_ok(*ts):
            ts = (_rows(x), _rows(dt), _dense(aneg), _rows(b_in), _rows(c_in), cu.contiguous(),
                  _dense(h0))
            if not torch.compiler.is_compiling():
                _native_packed._check_packed_scan("selective_scan_packed", *ts)
        return dispatch("packed_scan_fwd")(*ts, return_state, with_ckpt), ts

    @staticmethod
    def forward(ctx, x, dt, aneg, b_in, c_in, cu, h0, return_state):
        grad = any(ctx.needs_input_grad)
        (y, h_last, ckpt), ts = SelectiveScanPackedHIP.run(x, dt, aneg, b_in, c_in, cu, h0,
                                                           return_state, grad)
        if grad:
            ctx.save_for_backward(*ts, ckpt)
        ctx.set_materialize_grads(False)
        return (y, h_last) if return_state else y

    @staticmethod
    def backward(ctx, dy, dh_last=None):
        _once("selective_scan_packed")
        x, dt, aneg, b_in, c_in, cu, h0, ckpt = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(x)
        args = (x, dt, aneg, b_in, c_in, cu, h0, ckpt, dy, dh_last)
        if torch.compiler.is_compiling() or not _native_packed._scan_bwd_ok(*args):
            # (gradients of any layout; a saved-tensor hook may give another one, too)
            args = (_rows(x), _rows(dt), _dense(aneg), _rows(b_in), _rows(c_in), cu.contiguous(),
                    _dense(h0), _dense(ckpt), _rows(dy), _dense(dh_last))
            if not torch.compiler.is_compiling():
                _native_packed._check_packed_scan_bwd(*args)
        dx, ddt, da, db, dc, dh0 = dispatch("packed_scan_bwd")(*args)
        return dx, ddt, da, db, dc, None, dh0 if h0 is not None else None, None


class ConvSiluPackedHIP(torch.autograd.Function):
    """conv1d_silu_packed on the HIP kernels: (out, windows) or out."""

    @staticmethod
    def run(x, weight, bias, cu, window, return_window):
        """((out, windows), the operands as the kernels read them)."""
        ts = (x, weight, bias, cu, window)
        if torch.compiler.is_compiling() or not _native_packed._conv_ok(*ts):
            _conv_weight("conv1d_silu_packed", weight, x.shape[1])
            ts = (_rows(x), weight.reshape(weight.shape[0], -1).contiguous(), bias.contiguous(),
                  cu.contiguous(), window.contiguous() if window is not None else None)
            if not torch.compiler.is_compiling():
                _native_packed._check_packed_conv("conv1d_silu_packed", *ts)
        return dispatch("packed_conv_fwd")(*ts, return_window), ts

    @staticmethod
    def forward(ctx, x, weight, bias, cu, window, return_window):
        (out, last), ts = ConvSiluPackedHIP.run(x, weight, bias, cu, window, return_window)
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(*ts)
        ctx.wshape = weight.shape
        ctx.set_materialize_grads(False)
        return (out, last) if return_window else out

    @staticmethod
    def backward(ctx, dout, dlast=None):
        _once("conv1d_silu_packed")
        x, w, bias, cu, window = ctx.saved_tensors
        if dout is None:
            dout = torch.zeros_like(x)
        args = (x, w, bias, cu, window, dout, dlast)
        if torch.compiler.is_compiling() or not _native_packed._conv_bwd_ok(*args):
            args = (_rows(x), w.reshape(w.shape[0], -1).contiguous(), bias.contiguous(),
                    cu.contiguous(), window.contiguous() if window is not None else None,
                    _rows(dout),
                    dlast.contiguous() if dlast is not None else None)
            if not torch.compiler.is_compiling():
                _native_packed._check_packed_conv_bwd(*args)
        dx, dw, db, dwin = dispatch("packed_conv_bwd")(*args)
        return (dx, dw.view(ctx.wshape), db, None, dwin if window is not None else None, None)


def _conv_weight(what: str, weight: torch.Tensor, d: int) -> None:
    if not (weight.dim() == 2 or (weight.dim() == 3 and weight.shape[1] == 1)) \
            or weight.shape[0] != d:
        raise ValueError(f"{what}: weight must be ({d}, 1, K) or ({d}, K); got "
                         f"{tuple(weight.shape)}")


def conv1d_silu_packed(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
                       cu_seqlens: torch.Tensor, window: Optional[torch.Tensor] = None,
                       return_window: bool = False):
    """silu(causal depthwise conv1d(x)) of each of S packed sequences.

    x (L, D), its rows at any stride below 2^18 (as the x half of the block's in_proj output);
    weight (D, 1, K) or (D, K) and bias (D) of x's type or both float32, K up to 8; cu_seqlens
    (S + 1) int32 or int64, from 0 up, none above L. window (S, D, K - 1): the inputs before
    each sequence, oldest first (zeros without). Returns the (L, D) output, zeros in the
    rows behind the last sequence, and with return_window the (S, D, K - 1) last inputs of each,
    window's among them where it has fewer rows. Sums are float32; the gradients (x, weight, bias,
    window) are summed in a fixed order."""
    what = "conv1d_silu_packed"
    _hip(what, x, weight, bias, cu_seqlens, window)
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be (L, D); got {tuple(x.shape)}")
    if _records(x, weight, bias, window):
        return ConvSiluPackedHIP.apply(x, weight, bias, cu_seqlens, window, return_window)
    out = ConvSiluPackedHIP.run(x, weight, bias, cu_seqlens, window, return_window)[0]
    return out if return_window else out[0]


def selective_scan_packed(x: torch.Tensor, dt: torch.Tensor, aneg: torch.Tensor,
                          b_in: torch.Tensor, c_in: torch.Tensor, cu_seqlens: torch.Tensor,
                          h0: Optional[torch.Tensor] = None, return_state: bool = False):
    """selective_scan of each of S packed sequences.

    x, dt (L, D), B, C (L, N), of one type (float32, bfloat16, float16), rows at any stride
    below 2^18; Aneg (D, N) float32, N up to 64; cu_seqlens (S + 1) int32 or int64, from 0
    up, none above L. h0 (S, D, N) float32: the states before each sequence (zeros
    without). Returns y (L, D), zeros in the rows behind the last sequence, and with
    return_state the (S, D, N) float32 states behind each sequence (h0's for an empty one).
    An Aneg of +inf is a state that keeps nothing of the row before. The gradients (x, dt,
    Aneg, B, C, h0) are summed in a fixed order. For them the states at every eighth row
    are kept, L D N / 2 bytes. While it runs, a call of more than 64 rows holds some
    8 P D N bytes, its backward 12 P D N + L D N / 16, P pieces of 16 to 1024 rows, L over their
    length and one a sequence."""
    what = "selective_scan_packed"
    _hip(what, x, dt, aneg, b_in, c_in, cu_seqlens, h0)
    for name, t in (("x", x), ("dt", dt), ("B", b_in), ("C", c_in)):
        if t.dim() != 2:
            raise ValueError(f"{what}: {name} must have two dimensions; got {tuple(t.shape)}")
    if _records(x, dt, aneg, b_in, c_in, h0):
        return SelectiveScanPackedHIP.apply(x, dt, aneg, b_in, c_in, cu_seqlens, h0, return_state)
    y, h_last, _ = SelectiveScanPackedHIP.run(x, dt, aneg, b_in, c_in, cu_seqlens, h0,
                                              return_state, False)[0]
    return (y, h_last) if return_state else y


def _in_place(what: str, name: str, t: torch.Tensor) -> None:
    if not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{what} updates {name} in place; it must be contiguous and 16-byte "
                         "aligned")


def _no_grad(what: str, *ts: torch.Tensor) -> None:
    if _records(*ts) and not torch.compiler.is_compiling():
        raise RuntimeError(f"{what} updates its pool in place and has no gradients; call it "
                           "under torch.no_grad()")


def conv1d_silu_step(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
                     window: torch.Tensor, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of conv1d_silu for each row of x (R, D), in place on a pool of windows.

    window (P, D, K - 1) of x's type holds the last K - 1 inputs of P requests, oldest
    first; row r advances entry slots[r] (int32 or int64; without slots entry r).
    A slot below 0 is padding: its row gives 0. A slot past the pool, or one that an earlier
    row has too, gives a row of NaN; neither changes an entry. weight and bias as for
    conv1d_silu_packed. Returns the (R, D) output. Not differentiable."""
    what = "conv1d_silu_step"
    if not torch.compiler.is_compiling() and not _records(x, weight, bias, window) \
            and _native_packed._conv_step_ok(x, weight, bias, window, slots):
        return dispatch("conv_step")(x, weight, bias, window, slots)
    _hip(what, x, weight, bias, window, slots)
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be (R, D); got {tuple(x.shape)}")
    _conv_weight(what, weight, x.shape[1])
    _no_grad(what, x, weight, bias, window)
    if not window.is_contiguous():
        raise ValueError(f"{what} updates window in place; it must be contiguous")
    args = (_rows(x),
            (weight if weight.dim() == 2 else weight.reshape(weight.shape[0], -1)).contiguous(),
            bias.contiguous(), window, slots.contiguous() if slots is not None else None)
    if not torch.compiler.is_compiling():
        _native_packed._check_conv_step(*args)
    return dispatch("conv_step")(*args)


def selective_state_step_slots(h: torch.Tensor, x: torch.Tensor, dt: torch.Tensor,
                               aneg: torch.Tensor, b_in: torch.Tensor, c_in: torch.Tensor,
                               slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One recurrent step of the scan for each of R rows, in place on a pool of states.

    h (P, D, N) float32 holds the states of P requests; row r of x, dt (R, D) and B, C
    (R, N) (float32, bfloat16 or float16) advances entry slots[r] (int32 or int64; without
    slots entry r), with padding and slots that do not hold as in conv1d_silu_step. Returns y (R, D)
    of x's type. Not differentiable."""
    what = "selective_state_step_slots"
    if not torch.compiler.is_compiling() and not _records(h, x, dt, aneg, b_in, c_in) \
            and _native_packed._state_step_ok(h, x, dt, aneg, b_in, c_in, slots):
        return dispatch("state_step")(h, x, dt, aneg, b_in, c_in, slots)
    _hip(what, h, x, dt, aneg, b_in, c_in, slots)
    _no_grad(what, h, x, dt, aneg, b_in, c_in)
    if not torch.compiler.is_compiling():
        _in_place(what, "h", h)
    args = (h, _rows(x), _rows(dt), _dense(aneg), _rows(b_in), _rows(c_in),
            slots.contiguous() if slots is not None else None)
    if not torch.compiler.is_compiling():
        _native_packed._check_state_step(*args)
    return dispatch("state_step")(*args)
