"""What the head's losses refuse, on the CPU: the public functions' checks, the
registered ops', and the C entries' (fake device addresses that fail before any
use; only on hosts without a GPU, so that none can reach a launch)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mamba_metal_scan_amd import _native, distill_loss, linear_cross_entropy, linear_distill_loss
from mamba_metal_scan_amd._native import HipScanError

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device addresses")
A = ctypes.c_void_p(0x7F0000001000)
MIS = ctypes.c_void_p(0x7F0000001004)
EINVAL = 1


def test_cpu_tensors_are_refused():
    h, w, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    values, ids = torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm device"):
        linear_cross_entropy(h, w, t)
    with pytest.raises(RuntimeError, match="ROCm device"):
        linear_distill_loss(h, w, values, ids)
    with pytest.raises(RuntimeError, match="ROCm device"):
        distill_loss(torch.zeros(4, 5), values, ids)
    ops = torch.ops.mamba_hip
    with pytest.raises(HipScanError, match="ROCm device"):
        ops.linear_xent_fwd(h, w, t, -100, 1)
    with pytest.raises(HipScanError, match="ROCm device"):
        ops.linear_distill_fwd(h, w, values, ids, 1.0, 1)
    with pytest.raises(HipScanError, match="ROCm device"):
        ops.distill_fwd(torch.zeros(4, 5), values, ids, 1.0, 1)


def test_shapes_and_types_are_checked(monkeypatch):
    from mamba_metal_scan_amd import head
    monkeypatch.setattr(head, "_hip", lambda *a: None)   # (the device check comes first)
    h, w, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    values, ids = torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64)
    for args, kw, match in (
            ((h, w, t[:3]), {}, "targets"), ((h, w, t.float()), {}, "targets"),
            ((h, w, t), {"reduction": "avg"}, "reduction"),
            ((h, w, t), {"logits_bytes": -1}, "logits_bytes"),
            ((h, w, t), {"logits_bytes": 1e9}, "logits_bytes"),
            ((h, torch.zeros(5, 9), t), {}, "weight"), ((h, torch.zeros(0, 8), t), {}, "empty"),
            ((torch.zeros(4, 0), torch.zeros(5, 0), t), {}, "empty"),
            ((h, w.double(), t), {}, "float32, bfloat16"),
            ((h.double(), w.double(), t), {}, "float32, bfloat16")):
        with pytest.raises((ValueError, RuntimeError), match=match):
            linear_cross_entropy(*args, **kw)
    for v, i, kw, match in (
            (values, ids[:3], {}, "teacher"), (values[:, :1], ids, {}, "teacher"),
            (values[:, :0], ids[:, :0], {}, "words per row"),
            (torch.zeros(4, 1025), torch.zeros(4, 1025).long(), {}, "words per row"),
            (values, ids.float(), {}, "integers"), (values.long(), ids, {}, "floating"),
            (values, ids, {"temperature": 0.0}, "temperature"),
            (values, ids, {"temperature": float("nan")}, "temperature"),
            (values, ids, {"temperature": float("inf")}, "temperature"),
            (values, ids, {"reduction": "max"}, "reduction")):
        with pytest.raises((ValueError, RuntimeError), match=match):
            linear_distill_loss(h, w, v, i, **kw)
        with pytest.raises((ValueError, RuntimeError), match=match):
            distill_loss(torch.zeros(4, 50), v, i, **kw)
    with pytest.raises(ValueError, match="logits"):
        distill_loss(torch.zeros(4, 0), values, ids)
    with pytest.raises(RuntimeError, match="float32, bfloat16"):
        distill_loss(torch.zeros(4, 9).double(), values, ids)


def _err():
    return _native.library().mhs_last_error().decode()


def _xent_fwd(dtype=1, hidden=A, ldh=64, weight=A, ldw=64, targets=A, rows=4, vocab=50, dim=64,
              reduction=1, loss=A, logits=None, ws=A, nbytes=None):
    lib = _native.library()
    if nbytes is None:
        nbytes = lib.mhs_linear_xent_fwd_workspace_bytes(1, 4, 50, 64)
    return lib.mhs_linear_xent_fwd(dtype, hidden, ldh, weight, ldw, targets, A, A, A, logits, A,
                                   loss, A,
                                   rows, vocab, dim, -100, reduction, ws, nbytes, None)


@no_gpu
@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(reduction=3), "reduction"), (dict(rows=-1), "rows"),
    (dict(vocab=0), "vocab"), (dict(dim=60), "multiple of 8"), (dict(ldh=60), "strides"),
    (dict(ldh=65), "strides"), (dict(ldw=1 << 21), "strides"), (dict(hidden=MIS), "aligned"),
    (dict(weight=None), "null"), (dict(hidden=None), "null"), (dict(targets=None), "null"),
    (dict(loss=None), "null"), (dict(nbytes=16), "too small"), (dict(ws=None), "too small"),
    (dict(ws=MIS), "256-byte"), (dict(logits=MIS), "aligned"),
    (dict(rows=1 << 30, vocab=1 << 30), "too large")])
def test_cross_entropy_entry_refuses(kw, match):
    assert _xent_fwd(**kw) == EINVAL
    assert match in _err(), _err()


@no_gpu
def test_backward_entries_refuse():
    lib = _native.library()
    nbytes = lib.mhs_linear_xent_bwd_workspace_bytes(1, 4, 50, 64)

    def bwd(upstream=A, count=A, dh=A, nbytes=nbytes, ws=A, reduction=1, logits=None):
        return lib.mhs_linear_xent_bwd(1, A, 64, A, 64, A, A, A, A, logits, upstream, count,
                                       dh, A, 4, 50, 64, reduction, ws, nbytes, None)
    for kw, match in ((dict(upstream=None), "null"), (dict(count=None), "null"),
                      (dict(dh=MIS), "aligned"), (dict(nbytes=nbytes - 1), "too small"),
                      (dict(ws=MIS), "256-byte"), (dict(reduction=-1), "reduction"),
                      (dict(logits=MIS), "aligned")):
        assert bwd(**kw) == EINVAL and match in _err(), (kw, _err())

    def distill(top=4, temperature=1.0, q=A, teacher=A):
        return lib.mhs_linear_distill_fwd(1, A, 64, A, 64, teacher, A, A, A, q, A, None, A, A, A,
                                          4, 50, 64, top, temperature, 1, A, nbytes, None)
    for kw, match in ((dict(top=0), "words"), (dict(top=1025), "words"),
                      (dict(temperature=0.0), "temperature"),
                      (dict(temperature=float("nan")), "temperature"),
                      (dict(temperature=1e-45), "temperature"), (dict(q=None), "null"),
                      (dict(teacher=None), "null")):
        assert distill(**kw) == EINVAL and match in _err(), (kw, _err())


@no_gpu
def test_logits_entries_refuse():
    lib = _native.library()

    def fwd(dtype=0, logits=A, ld=50, rows=4, vocab=50, top=3, temperature=1.0, teacher=A, ws=A,
            nbytes=256, reduction=1):
        return lib.mhs_distill_fwd(dtype, logits, ld, teacher, A, A, A, A, A, A, A, rows, vocab,
                                   top, temperature, reduction, ws, nbytes, None)
    for kw, match in ((dict(dtype=-1), "dtype"), (dict(ld=49), "stride"), (dict(vocab=0), "vocab"),
                      (dict(logits=None), "null"), (dict(top=0), "words"),
                      (dict(temperature=-1.0), "temperature"), (dict(teacher=None), "null"),
                      (dict(logits=ctypes.c_void_p(0x7F0000001002)), "aligned"),
                      (dict(rows=20000, nbytes=16), "too small"), (dict(reduction=9), "reduction")):
        assert fwd(**kw) == EINVAL and match in _err(), (kw, _err())

    def bwd(logits=A, dlogits=ctypes.c_void_p(0x7F0000101000), count=A):
        return lib.mhs_distill_bwd(0, logits, 50, A, A, A, A, A, count, dlogits, 4, 50, 3, 1.0, 1,
                                   None)
    for kw, match in ((dict(dlogits=A), "alias"), (dict(dlogits=MIS), "aligned"),
                      (dict(count=None), "null"), (dict(dlogits=None), "null")):
        assert bwd(**kw) == EINVAL and match in _err(), (kw, _err())


def test_workspace_sizes():
    """Forward: 8 bytes per row and tile of the vocabulary (64 words for up to 16
    rows, 32 in fp32; above, 256, or 128 in fp32). Backward: the logits' gradient is bounded, a
    piece of the vocabulary; none for sizes that the calls reject."""
    lib = _native.library()
    fwd, bwd = lib.mhs_linear_xent_fwd_workspace_bytes, lib.mhs_linear_xent_bwd_workspace_bytes
    assert fwd(1, 8192, 32768, 640) == 8192 * 128 * 8
    assert fwd(0, 8192, 32768, 640) == 8192 * 256 * 8
    assert fwd(1, 4, 32768, 640) == 4 * 512 * 8
    assert fwd(1, 17, 32768, 640) == 17 * 128 * 8
    assert fwd(0, 32, 32768, 640) == 32 * 512 * 8
    whole = 8192 * 131072 * 2
    assert bwd(1, 8192, 131072, 64) < whole / 4
    assert bwd(1, 1, 131072, 640) < 2 << 20
    assert fwd(1, 8, 100, 60) == 0 and bwd(1, 8, 100, 60) == 0 and fwd(7, 8, 100, 64) == 0
    assert fwd(1, 0, 100, 64) > 0 and bwd(1, 0, 100, 64) > 0


def test_rule_of_kept_logits():
    """At most 1 GB of them; of 16-bit operands where that saves time."""
    def keeps(*a, most=1 << 30):
        return _native.keeps_logits(*a, most)
    f, b = torch.float32, torch.bfloat16
    assert keeps(8192, 32768, 640, f) and not keeps(8193, 32768, 640, f)
    assert keeps(256, 32768, 640, b) and not keeps(257, 32768, 640, b)
    assert keeps(2048, 131072, 2048, b) and not keeps(2049, 131072, 2048, b)
    assert keeps(0, 5, 8, f) and not keeps(1, 5, 8, f, most=0)
    assert keeps(4, 5, 8, f, most=80) and not keeps(4, 5, 8, f, most=79)


def test_fake_ops_have_the_kernels_shapes():
    """The shapes that tracing sees."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        h = torch.empty(6, 64, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(50, 64, device="cuda", dtype=torch.bfloat16)
        t = torch.empty(6, dtype=torch.int64, device="cuda")
        ids = torch.empty(6, 4, dtype=torch.int64, device="cuda")
        ops = torch.ops.mamba_hip
        loss, saved = ops.linear_xent_fwd(h, w, t, -100, 1)
        assert loss.shape == () and saved.dtype == torch.float32
        dh, dw = ops.linear_xent_bwd(loss, h, w, t, saved, 1, True, False)
        assert dh.shape == h.shape and dw.shape == (0,) and dh.dtype == h.dtype
        assert saved.shape == (4 + 6 * 4,)
        assert ops.linear_xent_fwd(h, w, t, -100, 1, True)[1].shape == (28 + 6 * 52,)
        kept = ops.linear_xent_fwd(h.float(), w.float(), t, -100, 1, True)[1]
        assert kept.shape == (28 + 50 * 8,)
        loss, saved = ops.linear_distill_fwd(h, w, ids.float(), ids, 1.0, 0)
        assert loss.shape == (6,)
        dh, dw = ops.linear_distill_bwd(loss, h, w, ids, saved, 1.0, 0, True, True)
        assert dw.shape == w.shape
        loss, saved = ops.distill_fwd(torch.empty(6, 50, device="cuda"), ids.float(), ids, 1.0, 2)
        assert ops.distill_bwd(loss, torch.empty(6, 50, device="cuda"), ids, saved, 1.0,
                               2).shape == (6, 50)
