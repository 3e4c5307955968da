"""The torch custom ops over packed sequences, tokens by slot and sampling: the
part of the library's binding (``_native.py``) that packed.py and sampling.py use.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._native import (HEAD_DTYPES, HipScanError, _check, _fp32, _need, _on, _on_one_device, _ptr,
                      _register, _shaped, _stream, library)

DTYPES = HEAD_DTYPES            # activations: the library's number of each type
MAX_TAPS = 8
MAX_STATE = 64
MAX_STRIDE = 1 << 18
CKPT = 8                        # rows between the scan's checkpoints
_INTS = (torch.int32, torch.int64)


def rows_ok(t: torch.Tensor) -> bool:
    """Whether the kernels read the 2-D t in place: its rows are dense, do not overlap,
    and lie less than 2^18 elements apart."""
    n, w = t.shape
    return ((w <= 1 or t.stride(1) == 1)
            and (n <= 1 or w <= t.stride(0) < MAX_STRIDE))


def _ld(t: torch.Tensor, rows: int, width: int) -> int:
    return t.stride(0) if rows > 1 else width


# Each check has a quick form first, a single expression over what usually holds, and only
# where that is false the one that names what is wrong (the checks were a third of a small
# call's host time: a conv step 15.8 us, 6.0 of them the check's).

def _like(t: torch.Tensor, shape, dtype, index: int) -> bool:
    """t has the shape, type and device, and rows that the kernels read."""
    return (t.shape == shape and t.dtype is dtype and t.get_device() == index and rows_ok(t))


def _f32(t: Optional[torch.Tensor], shape, index: int) -> bool:
    return t is None or (t.shape == shape and t.dtype is torch.float32
                         and t.get_device() == index and t.is_contiguous()
                         and not t.data_ptr() & 15)


def _ints(t: torch.Tensor, index: int) -> bool:
    return (t.dim() == 1 and t.dtype in _INTS and t.get_device() == index
            and t.is_contiguous())


def _act(what: str, x: torch.Tensor, **like: Optional[torch.Tensor]) -> None:
    """x (rows, D) and what is of its type, in rows that the kernels read."""
    _need(x.dim() == 2, what, f"x must be (rows, D); got {tuple(x.shape)}")
    for name, t in dict(x=x, **like).items():
        if t is None:
            continue
        if t.dtype != x.dtype or x.dtype not in DTYPES:
            raise HipScanError(f"{what}: {', '.join(['x', *like])} must all be float32, bfloat16 "
                               f"or float16; got {x.dtype}, {name} {t.dtype}")
        _need(t.dim() == 2 and rows_ok(t), what,
              f"{name} needs dense rows less than 2^18 elements apart; got strides {t.stride()} "
              f"for shape {tuple(t.shape)}")


def _dense16(what: str, **ts: Optional[torch.Tensor]) -> None:
    for name, t in ts.items():
        if t is not None and not (t.is_contiguous() and t.data_ptr() % 16 == 0):
            raise HipScanError(f"{what}: {name} must be contiguous and 16-byte aligned")


def _seqs(what: str, cu: torch.Tensor) -> int:
    """The number of sequences."""
    _need(cu.dim() == 1 and cu.numel() >= 1 and cu.dtype in _INTS and cu.is_contiguous(), what,
          "cu_seqlens must be a contiguous vector of int32 or int64, one number more than "
          f"sequences; got {cu.dtype} {tuple(cu.shape)}")
    return cu.numel() - 1


# ----------------------------------------------------------------- the scan

def _scan_ok(x, dt, aneg, b_in, c_in, cu, h0) -> bool:
    if x.dim() != 2 or aneg.dim() != 2 or x.dtype not in DTYPES:
        return False
    index, dtype, shape = x.get_device(), x.dtype, x.shape
    d, n = aneg.shape
    bc = (shape[0], n)
    return (index >= 0 and 1 <= n <= MAX_STATE and d >= 1 and shape[1] == d and rows_ok(x)
            and _like(dt, shape, dtype, index) and _like(b_in, bc, dtype, index)
            and _like(c_in, bc, dtype, index) and _f32(aneg, (d, n), index)
            and _ints(cu, index) and cu.shape[0] >= 1
            and _f32(h0, (cu.shape[0] - 1, d, n), index))


def _check_packed_scan(what: str, x, dt, aneg, b_in, c_in, cu, h0) -> None:
    if _scan_ok(x, dt, aneg, b_in, c_in, cu, h0):
        return
    _on_one_device(what, x, dt, aneg, b_in, c_in, cu, h0)
    _act(what, x, dt=dt, B=b_in, C=c_in)
    _need(aneg.dim() == 2, what, f"Aneg must be (D, N); got {tuple(aneg.shape)}")
    rows, d = x.shape
    n = aneg.shape[1]
    _need(1 <= n <= MAX_STATE and d >= 1, what,
          f"D must be at least 1 and N in [1, {MAX_STATE}]; got {d}, {n}")
    _shaped(what, "dt", dt, (rows, d))
    _shaped(what, "Aneg", aneg, (d, n))
    _shaped(what, "B", b_in, (rows, n))
    _shaped(what, "C", c_in, (rows, n))
    _shaped(what, "h0", h0, (_seqs(what, cu), d, n))
    _fp32(what, Aneg=aneg, h0=h0)
    _dense16(what, Aneg=aneg, h0=h0)


def _packed_scan_fwd_impl(x: torch.Tensor, dt: torch.Tensor, aneg: torch.Tensor,
                          b_in: torch.Tensor, c_in: torch.Tensor, cu: torch.Tensor,
                          h0: Optional[torch.Tensor], want_state: bool, with_ckpt: bool
                          ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, h_last, ckpt); the last two empty where not wanted."""
    rows, d = x.shape
    n, seqs = aneg.shape[1], cu.numel() - 1
    lib = library()
    y = x.new_empty((rows, d))
    h_last = aneg.new_empty((seqs, d, n) if want_state else (0,))
    ckpt = aneg.new_empty((lib.mhs_packed_ckpt_floats(rows, d, n) if with_ckpt else 0,))
    dev = x.device
    with _on(dev):
        nbytes = lib.mhs_packed_scan_workspace_bytes(seqs, rows, d, n, 0)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = lib.mhs_packed_scan_fwd(
            DTYPES[x.dtype], x.data_ptr(), _ld(x, rows, d), dt.data_ptr(),
            _ld(dt, rows, d), aneg.data_ptr(), b_in.data_ptr(), _ld(b_in, rows, n),
            c_in.data_ptr(), _ld(c_in, rows, n), cu.data_ptr(), cu.dtype == torch.int64,
            _ptr(h0), y.data_ptr(), h_last.data_ptr() if want_state else None,
            ckpt.data_ptr() if with_ckpt else None,
            seqs, rows, d, n, _ptr(ws), nbytes, _stream(dev))
    _check(rc, "mhs_packed_scan_fwd")
    return y, h_last, ckpt


packed_scan_fwd = _register(
    "packed_scan_fwd", _packed_scan_fwd_impl, (),
    lambda x, dt, aneg, b_in, c_in, cu, h0, want_state, with_ckpt:
    _check_packed_scan("packed_scan_fwd", x, dt, aneg, b_in, c_in, cu, h0))


@packed_scan_fwd.register_fake
def _packed_scan_fwd_fake(x, dt, aneg, b_in, c_in, cu, h0, want_state, with_ckpt):
    rows, d = x.shape
    n, seqs = aneg.shape[1], cu.shape[0] - 1
    return (x.new_empty((rows, d)), aneg.new_empty((seqs, d, n) if want_state else (0,)),
            aneg.new_empty((rows // CKPT * d * n if with_ckpt else 0,)))


def _packed_scan_bwd_impl(x: torch.Tensor, dt: torch.Tensor, aneg: torch.Tensor,
                          b_in: torch.Tensor, c_in: torch.Tensor, cu: torch.Tensor,
                          h0: Optional[torch.Tensor], ckpt: torch.Tensor, dy: torch.Tensor,
                          dh_last: Optional[torch.Tensor]
                          ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                     torch.Tensor, torch.Tensor]:
    """(dx, ddt, dAneg, dB, dC, dh0); the last empty without h0."""
    rows, d = x.shape
    n, seqs = aneg.shape[1], cu.numel() - 1
    lib = library()
    dx, ddt = x.new_empty((rows, d)), x.new_empty((rows, d))
    db, dc = x.new_empty((rows, n)), x.new_empty((rows, n))
    da = aneg.new_empty((d, n))
    dh0 = aneg.new_empty((seqs, d, n) if h0 is not None else (0,))
    dev = x.device
    with _on(dev):
        nbytes = lib.mhs_packed_scan_workspace_bytes(seqs, rows, d, n, 1)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = lib.mhs_packed_scan_bwd(
            DTYPES[x.dtype], x.data_ptr(), _ld(x, rows, d), dt.data_ptr(),
            _ld(dt, rows, d), aneg.data_ptr(), b_in.data_ptr(), _ld(b_in, rows, n),
            c_in.data_ptr(), _ld(c_in, rows, n), cu.data_ptr(), cu.dtype == torch.int64,
            _ptr(h0), ckpt.data_ptr(), dy.data_ptr(), _ld(dy, rows, d), _ptr(dh_last),
            dx.data_ptr(), ddt.data_ptr(), da.data_ptr(), db.data_ptr(),
            dc.data_ptr(), dh0.data_ptr() if h0 is not None else None, seqs, rows, d, n, _ptr(ws),
            nbytes, _stream(dev))
    _check(rc, "mhs_packed_scan_bwd")
    return dx, ddt, da, db, dc, dh0


def _scan_bwd_ok(x, dt, aneg, b_in, c_in, cu, h0, ckpt, dy, dh_last) -> bool:
    if not _scan_ok(x, dt, aneg, b_in, c_in, cu, h0):
        return False
    index = x.get_device()
    d, n = aneg.shape
    return (_like(dy, x.shape, x.dtype, index) and _f32(dh_last, (cu.shape[0] - 1, d, n), index)
            and _f32(ckpt, (x.shape[0] // CKPT * d * n,), index))


def _check_packed_scan_bwd(x, dt, aneg, b_in, c_in, cu, h0, ckpt, dy, dh_last) -> None:
    what = "packed_scan_bwd"
    if _scan_bwd_ok(x, dt, aneg, b_in, c_in, cu, h0, ckpt, dy, dh_last):
        return
    _check_packed_scan(what, x, dt, aneg, b_in, c_in, cu, h0)
    _on_one_device(what, x, ckpt, dy, dh_last)
    _act(what, x, dy=dy)
    rows, d = x.shape
    n = aneg.shape[1]
    _shaped(what, "dy", dy, (rows, d))
    _shaped(what, "dh_last", dh_last, (cu.numel() - 1, d, n))
    _shaped(what, "ckpt", ckpt, (rows // CKPT * d * n,))
    _fp32(what, ckpt=ckpt, dh_last=dh_last)
    _dense16(what, ckpt=ckpt, dh_last=dh_last)


packed_scan_bwd = _register("packed_scan_bwd", _packed_scan_bwd_impl, (), _check_packed_scan_bwd)


@packed_scan_bwd.register_fake
def _packed_scan_bwd_fake(x, dt, aneg, b_in, c_in, cu, h0, ckpt, dy, dh_last):
    rows, d = x.shape
    n = aneg.shape[1]
    return (x.new_empty((rows, d)), x.new_empty((rows, d)), aneg.new_empty((d, n)),
            x.new_empty((rows, n)), x.new_empty((rows, n)),
            aneg.new_empty((cu.shape[0] - 1, d, n) if h0 is not None else (0,)))


# ---------------------------------------------------------- the convolution

def _check_taps(what: str, x, w, bias) -> None:
    """w (D, K) and bias (D) of x's type, or both fp32."""
    _need(w.dim() == 2 and 1 <= w.shape[1] <= MAX_TAPS and x.shape[1] >= 1, what,
          f"w must be (D, K), D at least 1 and K in [1, {MAX_TAPS}]; got {tuple(w.shape)}")
    _shaped(what, "w", w, (x.shape[1], w.shape[1]))
    _shaped(what, "bias", bias, (x.shape[1],))
    _need(w.dtype == bias.dtype and w.dtype in (x.dtype, torch.float32), what,
          f"weight and bias must be of x's type {x.dtype} or both float32; got {w.dtype}, "
          f"{bias.dtype}")
    _need(w.is_contiguous() and bias.is_contiguous(), what, "weight and bias must be contiguous")


def _taps_ok(x, w, bias, index: int) -> bool:
    """(w (D, K), or (D, 1, K) as nn.Conv1d holds it: the same numbers in memory)"""
    if x.dim() != 2 or x.dtype not in DTYPES or not rows_ok(x):
        return False
    shape = w.shape
    if len(shape) != 2 and (len(shape) != 3 or shape[1] != 1):
        return False
    d, k = shape[0], shape[-1]
    return (index >= 0 and d >= 1 and 1 <= k <= MAX_TAPS and x.shape[1] == d
            and (w.dtype is x.dtype or w.dtype is torch.float32) and w.get_device() == index
            and w.is_contiguous() and bias.shape == (d,) and bias.dtype is w.dtype
            and bias.get_device() == index and bias.is_contiguous())


def _window_ok(t, x, entries: int, taps: int, index: int) -> bool:
    return t is None or (t.shape == (entries, x.shape[1], taps - 1) and t.dtype is x.dtype
                         and t.get_device() == index and t.is_contiguous())


def _conv_ok(x, w, bias, cu, window) -> bool:
    index = x.get_device()
    return (_taps_ok(x, w, bias, index) and _ints(cu, index) and cu.shape[0] >= 1
            and _window_ok(window, x, cu.shape[0] - 1, w.shape[-1], index))


def _check_packed_conv(what: str, x, w, bias, cu, window) -> None:
    if _conv_ok(x, w, bias, cu, window):
        return
    _on_one_device(what, x, w, bias, cu, window)
    _act(what, x)
    _check_taps(what, x, w, bias)
    _shaped(what, "window", window, (_seqs(what, cu), x.shape[1], w.shape[1] - 1))
    _need(window is None or (window.dtype == x.dtype and window.is_contiguous()), what,
          f"window must be contiguous and of x's type {x.dtype}")


def _packed_conv_fwd_impl(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, cu: torch.Tensor,
                          window: Optional[torch.Tensor], want_window: bool
                          ) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, the windows behind the sequences or an empty tensor)."""
    rows, d = x.shape
    k, seqs = w.shape[-1], cu.numel() - 1
    out = x.new_empty((rows, d))
    last = x.new_empty((seqs, d, k - 1) if want_window else (0,))
    dev = x.device
    with _on(dev):
        rc = library().mhs_packed_conv_fwd(
            DTYPES[x.dtype], x.data_ptr(), _ld(x, rows, d), w.data_ptr(), bias.data_ptr(),
            w.dtype == torch.float32, cu.data_ptr(), cu.dtype == torch.int64, _ptr(window),
            out.data_ptr(), last.data_ptr() if want_window else None, seqs, rows, d, k,
            _stream(dev))
    _check(rc, "mhs_packed_conv_fwd")
    return out, last


packed_conv_fwd = _register(
    "packed_conv_fwd", _packed_conv_fwd_impl, (),
    lambda x, w, bias, cu, window, want_window:
    _check_packed_conv("packed_conv_fwd", x, w, bias, cu, window))


@packed_conv_fwd.register_fake
def _packed_conv_fwd_fake(x, w, bias, cu, window, want_window):
    rows, d = x.shape
    return (x.new_empty((rows, d)),
            x.new_empty((cu.shape[0] - 1, d, w.shape[-1] - 1) if want_window else (0,)))


def _packed_conv_bwd_impl(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, cu: torch.Tensor,
                          window: Optional[torch.Tensor], dout: torch.Tensor,
                          dlast: Optional[torch.Tensor]
                          ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dw, dbias, dwindow); the last empty without a window."""
    rows, d = x.shape
    k, seqs = w.shape[-1], cu.numel() - 1
    lib = library()
    dx, dw, db = x.new_empty((rows, d)), torch.empty_like(w), torch.empty_like(bias)
    dwin = x.new_empty((seqs, d, k - 1) if window is not None else (0,))
    dev = x.device
    with _on(dev):
        nbytes = lib.mhs_packed_conv_bwd_workspace_bytes(seqs, rows, d, k)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = lib.mhs_packed_conv_bwd(
            DTYPES[x.dtype], x.data_ptr(), _ld(x, rows, d), w.data_ptr(), bias.data_ptr(),
            w.dtype == torch.float32, cu.data_ptr(), cu.dtype == torch.int64, _ptr(window),
            dout.data_ptr(), _ld(dout, rows, d), _ptr(dlast), dx.data_ptr(), dw.data_ptr(),
            db.data_ptr(), dwin.data_ptr() if window is not None else None, seqs, rows, d, k,
            ws.data_ptr(), nbytes, _stream(dev))
    _check(rc, "mhs_packed_conv_bwd")
    return dx, dw, db, dwin


def _conv_bwd_ok(x, w, bias, cu, window, dout, dlast) -> bool:
    return (_conv_ok(x, w, bias, cu, window) and _like(dout, x.shape, x.dtype, x.get_device())
            and _window_ok(dlast, x, cu.shape[0] - 1, w.shape[-1], x.get_device()))


def _check_packed_conv_bwd(x, w, bias, cu, window, dout, dlast) -> None:
    what = "packed_conv_bwd"
    if _conv_bwd_ok(x, w, bias, cu, window, dout, dlast):
        return
    _check_packed_conv(what, x, w, bias, cu, window)
    _on_one_device(what, x, dout, dlast)
    _act(what, x, dout=dout)
    _shaped(what, "dout", dout, x.shape)
    _shaped(what, "dlast", dlast, (cu.numel() - 1, x.shape[1], w.shape[1] - 1))
    _need(dlast is None or (dlast.dtype == x.dtype and dlast.is_contiguous()), what,
          f"dlast must be contiguous and of x's type {x.dtype}")


packed_conv_bwd = _register("packed_conv_bwd", _packed_conv_bwd_impl, (), _check_packed_conv_bwd)


@packed_conv_bwd.register_fake
def _packed_conv_bwd_fake(x, w, bias, cu, window, dout, dlast):
    return (x.new_empty(x.shape), torch.empty_like(w), torch.empty_like(bias),
            x.new_empty((cu.shape[0] - 1, x.shape[1], w.shape[-1] - 1) if window is not None
                        else (0,)))


# ------------------------------------------------------------ tokens by slot

def _check_slots(what: str, slots, rows: int, pool: int) -> None:
    if slots is None:
        _need(rows <= pool, what, f"{rows} rows without slots need as many entries; got {pool}")
    else:
        _need(slots.dim() == 1 and slots.numel() == rows and slots.dtype in _INTS
              and slots.is_contiguous(), what,
              f"slots must be a contiguous int32 or int64 vector of {rows} numbers; got "
              f"{slots.dtype} {tuple(slots.shape)}")


def _slots_ok(slots, rows: int, pool: int, index: int) -> bool:
    return rows <= pool if slots is None else _ints(slots, index) and slots.shape[0] == rows


def _conv_step_ok(x, w, bias, window, slots) -> bool:
    index = x.get_device()
    return (_taps_ok(x, w, bias, index) and window.dim() == 3
            and _window_ok(window, x, window.shape[0], w.shape[-1], index)
            and _slots_ok(slots, x.shape[0], window.shape[0], index))


def _check_conv_step(x, w, bias, window, slots) -> None:
    what = "conv_step"
    if _conv_step_ok(x, w, bias, window, slots):
        return
    _on_one_device(what, x, w, bias, window, slots)
    _act(what, x)
    _check_taps(what, x, w, bias)
    _need(window.dim() == 3 and window.dtype == x.dtype and window.is_contiguous(), what,
          f"window must be contiguous (entries, D, K - 1) of x's type {x.dtype}; got "
          f"{window.dtype} {tuple(window.shape)}")
    _shaped(what, "window", window, (window.shape[0], x.shape[1], w.shape[1] - 1))
    _check_slots(what, slots, x.shape[0], window.shape[0])


def _conv_step_impl(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, window: torch.Tensor,
                    slots: Optional[torch.Tensor]) -> torch.Tensor:
    """out (rows, D); window's entries advanced in place."""
    rows, d = x.shape
    out = x.new_empty((rows, d))
    dev = x.device
    with _on(dev):
        rc = library().mhs_conv_step(
            DTYPES[x.dtype], x.data_ptr(), _ld(x, rows, d), w.data_ptr(), bias.data_ptr(),
            w.dtype == torch.float32, window.data_ptr(), _ptr(slots),
            slots is not None and slots.dtype == torch.int64, out.data_ptr(), rows,
            window.shape[0], d, w.shape[-1], _stream(dev))
    _check(rc, "mhs_conv_step")
    return out


conv_step = _register("conv_step", _conv_step_impl, ("window",), _check_conv_step)


@conv_step.register_fake
def _conv_step_fake(x, w, bias, window, slots):
    return x.new_empty(x.shape)


def _state_step_ok(h, x, dt, aneg, b_in, c_in, slots) -> bool:
    if x.dim() != 2 or h.dim() != 3 or x.dtype not in DTYPES:
        return False
    index, dtype, shape = x.get_device(), x.dtype, x.shape
    pool, d, n = h.shape
    bc = (shape[0], n)
    return (index >= 0 and 1 <= n <= MAX_STATE and d >= 1 and shape[1] == d and rows_ok(x)
            and _like(dt, shape, dtype, index) and _like(b_in, bc, dtype, index)
            and _like(c_in, bc, dtype, index) and _f32(aneg, (d, n), index)
            and _f32(h, (pool, d, n), index) and _slots_ok(slots, shape[0], pool, index))


def _check_state_step(h, x, dt, aneg, b_in, c_in, slots) -> None:
    what = "state_step"
    if _state_step_ok(h, x, dt, aneg, b_in, c_in, slots):
        return
    _on_one_device(what, h, x, dt, aneg, b_in, c_in, slots)
    _act(what, x, dt=dt, B=b_in, C=c_in)
    _need(h.dim() == 3, what, f"h must be (entries, D, N); got {tuple(h.shape)}")
    pool, d, n = h.shape
    rows = x.shape[0]
    _need(1 <= n <= MAX_STATE and d >= 1, what,
          f"D must be at least 1 and N in [1, {MAX_STATE}]; got {d}, {n}")
    for name, t, shape in (("x", x, (rows, d)), ("dt", dt, (rows, d)), ("Aneg", aneg, (d, n)),
                           ("B", b_in, (rows, n)), ("C", c_in, (rows, n))):
        _shaped(what, name, t, shape)
    _fp32(what, h=h, Aneg=aneg)
    _dense16(what, h=h, Aneg=aneg)
    _check_slots(what, slots, rows, pool)


def _state_step_impl(h: torch.Tensor, x: torch.Tensor, dt: torch.Tensor, aneg: torch.Tensor,
                     b_in: torch.Tensor, c_in: torch.Tensor, slots: Optional[torch.Tensor]
                     ) -> torch.Tensor:
    """y (rows, D); h's entries advanced in place."""
    rows, d = x.shape
    n = h.shape[2]
    y = x.new_empty((rows, d))
    dev = x.device
    with _on(dev):
        rc = library().mhs_state_step(
            DTYPES[x.dtype], h.data_ptr(), x.data_ptr(), _ld(x, rows, d), dt.data_ptr(),
            _ld(dt, rows, d), aneg.data_ptr(), b_in.data_ptr(), _ld(b_in, rows, n),
            c_in.data_ptr(), _ld(c_in, rows, n), _ptr(slots),
            slots is not None and slots.dtype == torch.int64, y.data_ptr(), rows, h.shape[0], d,
            n, _stream(dev))
    _check(rc, "mhs_state_step")
    return y


state_step = _register("state_step", _state_step_impl, ("h",), _check_state_step)


@state_step.register_fake
def _state_step_fake(h, x, dt, aneg, b_in, c_in, slots):
    return x.new_empty(x.shape)


# ----------------------------------------------------------------- sampling

def _vector(t, rows: int, index: int) -> bool:
    return t is None or (t.shape == (rows,) and t.dtype is torch.float32
                         and t.get_device() == index and t.is_contiguous())


def _sample_ok(logits, uniform, temperature, top_k, top_p, min_p, values_f) -> bool:
    if logits.dim() != 2 or logits.dtype not in DTYPES:
        return False
    rows, vocab = logits.shape
    index = logits.get_device()
    return (index >= 0 and vocab >= 1 and (vocab == 1 or logits.stride(1) == 1)
            and (rows <= 1 or logits.stride(0) >= vocab) and len(values_f) == 3
            and uniform is not None and _vector(uniform, rows, index)
            and _vector(temperature, rows, index) and _vector(top_p, rows, index)
            and _vector(min_p, rows, index)
            and (top_k is None or (_ints(top_k, index) and top_k.shape[0] == rows)))


def _check_sample(logits, uniform, temperature, top_k, top_p, min_p, values_f, value_k) -> None:
    what = "sample"
    if _sample_ok(logits, uniform, temperature, top_k, top_p, min_p, values_f):
        return
    _on_one_device(what, logits, uniform, temperature, top_k, top_p, min_p)
    _need(logits.dim() == 2 and logits.shape[1] >= 1 and logits.dtype in DTYPES, what,
          "logits must be (rows, vocab) in float32, bfloat16 or float16; got "
          f"{logits.dtype} {tuple(logits.shape)}")
    rows, vocab = logits.shape
    _need((vocab <= 1 or logits.stride(1) == 1) and (rows <= 1 or logits.stride(0) >= vocab), what,
          f"logits need contiguous rows; got strides {logits.stride()}")
    for name, t, dtypes in (("uniform", uniform, (torch.float32,)),
                            ("temperature", temperature, (torch.float32,)),
                            ("top_k", top_k, _INTS), ("top_p", top_p, (torch.float32,)),
                            ("min_p", min_p, (torch.float32,))):
        _need(t is None or (t.shape == (rows,) and t.dtype in dtypes and t.is_contiguous()), what,
              f"{name} must be a contiguous vector of {rows} {dtypes[0]}")
    _need(len(values_f) == 3, what, "three values: temperature, top_p, min_p")


def _sample_impl(logits: torch.Tensor, uniform: torch.Tensor, temperature: Optional[torch.Tensor],
                 top_k: Optional[torch.Tensor], top_p: Optional[torch.Tensor],
                 min_p: Optional[torch.Tensor], values_f: list[float], value_k: int
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens, log-probabilities); settings of the rows, or where None the values."""
    rows, vocab = logits.shape
    lib = library()
    dev = logits.device
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logps = torch.empty(rows, dtype=torch.float32, device=dev)
    with _on(dev):
        nbytes = lib.mhs_sample_workspace_bytes(rows, vocab, top_k is not None, value_k)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = lib.mhs_sample(
            DTYPES[logits.dtype], logits.data_ptr(), _ld(logits, rows, vocab), uniform.data_ptr(),
            _ptr(temperature), values_f[0], _ptr(top_k),
            top_k is not None and top_k.dtype == torch.int64, value_k, _ptr(top_p), values_f[1],
            _ptr(min_p), values_f[2], tokens.data_ptr(), logps.data_ptr(), rows, vocab, _ptr(ws),
            nbytes, _stream(dev))
    _check(rc, "mhs_sample")
    return tokens, logps


sample = _register("sample", _sample_impl, (), _check_sample)


@sample.register_fake
def _sample_fake(logits, uniform, temperature, top_k, top_p, min_p, values_f, value_k):
    rows = logits.shape[0]
    return (torch.empty(rows, dtype=torch.int64, device=logits.device),
            torch.empty(rows, dtype=torch.float32, device=logits.device))
