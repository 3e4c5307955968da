"""The cut of packed sequences into pieces, restated on the host: the rows, checkpoints, carries and
windows that the kernels index for any cu_seqlens, lengths or not, lie inside their tensors; of
lengths every row has one piece, every piece a number and every checkpoint an entry of its own."""
from __future__ import annotations

import random

import pytest

CKPT = 8          # rows between checkpoints (kCkpt)
CONV_PIECE = 16   # rows of a piece of the conv (kConvPiece, kConvBackPiece)


def at(cu, total, s):                                   # cu_at
    return max(0, min(cu[s], total))


def find_piece(cu, total, tc, p):
    """(seq, begin, j, t0, len, last), or None: the device's search, 64 probes a round."""
    nseq = len(cu) - 1
    lo, hi, rounds = 0, nseq + 1, 0
    while hi - lo > 1:
        rounds += 1
        assert rounds <= 8
        step = (hi - lo + 63) // 64
        n = sum(1 for lane in range(64)
                if lo + lane * step < hi
                and at(cu, total, lo + lane * step) // tc + lo + lane * step <= p)
        if n == 0:
            break
        lo += (n - 1) * step
        hi = min(hi, lo + step)
    assert 0 <= lo <= nseq
    b = at(cu, total, lo)
    e = total if lo == nseq else max(b, at(cu, total, lo + 1))
    j = p - (b // tc + lo)
    if j < 0 or (j > 0 and b + j * tc >= e):
        return None
    t0 = b + j * tc
    n = min(tc, e - t0)
    return lo, b, j, t0, n, t0 + n >= e


def pieces(cu, total, tc):
    """All numbers' pieces, as the grid has them."""
    for p in range(total // tc + len(cu) - 1 + 1):
        yield p, find_piece(cu, total, tc, p)


def check_in_bounds(cu, total, tc, taps):
    nseq, count = len(cu) - 1, total // tc + len(cu)
    for p, piece in pieces(cu, total, tc):
        if piece is None:
            continue
        seq, begin, j, t0, n, last = piece
        assert 0 <= seq <= nseq and 0 <= begin <= t0 and 0 <= n <= tc and t0 + n <= total
        for step in range(0, n, CKPT):                  # the forward's stores, the backward's loads
            if j > 0 or step > 0:
                entry = begin // CKPT + j * (tc // CKPT) + step // CKPT - 1
                assert 0 <= entry < total // CKPT
        if seq == nseq:
            continue
        # the conv: what is before the piece's first row, and behind its last in the backward
        for t in range(t0 - taps + 1, t0):
            if t < begin:
                assert 0 <= taps - 1 - (begin - t) < taps - 1
            else:
                assert 0 <= t < total
        end = t0 + n if last else max(at(cu, total, seq + 1), begin)
        assert begin <= end <= total
        for i in range(n + taps - 1):
            t = t0 + i
            r = t - taps + 1
            if t < end:
                assert 0 <= t < total
            if end - (taps - 1) <= r < end:
                assert 0 <= r - (end - (taps - 1)) < taps - 1
            if r >= t0:
                assert r < t0 + n
            elif j == 0:
                assert 0 <= r - (begin - (taps - 1)) < taps - 1
    for s in range(nseq):                               # the fold
        b = at(cu, total, s)
        n = max(1, (max(b, at(cu, total, s + 1)) - b + tc - 1) // tc)
        assert 0 <= b // tc + s and b // tc + s + n - 1 < count


LIMITS = [([0, 50, 20, 100], 100), ([-5, 50, 200], 100), ([90, 10, 95], 100), ([0, 1 << 30], 100),
          ([100, 100, 100, 0], 100), ([0, -(1 << 62), 1 << 62], 100), ([7], 100), ([0], 0),
          ([0, 0, 0], 0), ([5, 5], 3), ([3, 2, 1, 0], 3)]


@pytest.mark.parametrize("tc", [16, 32, 48, 160, 1024])
def test_numbers_that_are_no_lengths(tc):
    rng = random.Random(tc)
    cases = list(LIMITS)
    for _ in range(150):
        total = rng.choice([0, 1, 15, 16, 17, 100, 1000, 3001])
        nseq = rng.choice([0, 1, 2, 5, 63, 64, 65, 200])
        wide = rng.choice([total, total + 40, 10 * total + 7, 1 << 33])
        cases.append(([rng.randint(-wide, wide) for _ in range(nseq + 1)], total))
    for cu, total in cases:
        check_in_bounds(cu, total, tc, rng.choice([1, 2, 4, 8]))


@pytest.mark.parametrize("tc", [16, 32, 48, 160, 1024])
def test_lengths_cover_every_row_once(tc):
    rng = random.Random(tc)
    for _ in range(120):
        nseq = rng.choice([0, 1, 2, 5, 63, 64, 65, 300])
        top = rng.choice([1, 3, 17, 100, 700])
        cu = [0]
        for _ in range(nseq):
            cu.append(cu[-1] + rng.choice([0, 1, rng.randint(0, top), top]))
        total = cu[-1] + rng.choice([0, 1, 37])
        check_in_bounds(cu, total, tc, 4)
        rows, ends, entries = [0] * total, [0] * nseq, set()
        for p, piece in pieces(cu, total, tc):
            if piece is None:
                continue
            seq, begin, j, t0, n, last = piece
            assert begin == cu[seq] and t0 == begin + j * tc
            if seq < nseq:
                assert t0 + n <= cu[seq + 1] and last == (t0 + n == cu[seq + 1])
                ends[seq] += last
                for step in range(0, n, CKPT):
                    if j > 0 or step > 0:
                        entry = begin // CKPT + j * (tc // CKPT) + step // CKPT - 1
                        assert entry not in entries
                        entries.add(entry)
            for t in range(t0, t0 + n):
                rows[t] += 1
        assert all(r == 1 for r in rows) and all(e == 1 for e in ends)
