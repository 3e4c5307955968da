"""The order of what a stream of product tiles does with its slots of LDS (mm_stream:
what a tile's epilogue needs beside its sums), on the CPU: the constants are the
sources', the order of loads, waits and reads is written down here."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "mamba_metal_scan_amd" / "csrc"


def _constants():
    src = (CSRC / "mhs_mm16.hpp").read_text()
    stages = int(re.search(r"constexpr int kMmStages = (\d+);", src).group(1))
    slots = re.search(r"constexpr int kMmSlots = kMmStages \+ (\d+);", src)
    return stages, stages + int(slots.group(1)) if slots else 2


def _overwritten(tiles: int, nk: int, stages: int, slots: int) -> list[tuple[int, int]]:
    """(tile, the tile whose loads came into its slot before its epilogue read it, or
    with no barrier after that reading) of one block's stream of `tiles` tiles of nk k
    tiles: every k tile is one wait and barrier, then the loads of the k tile `stages`
    further, with a tile's first the slot's; the epilogue follows a tile's last."""
    bad, held, read_at = [], {}, {}
    barrier = 0
    loaded = [(t, k) for t in range(tiles) for k in range(nk)]
    def load(i):
        if i >= len(loaded) or loaded[i][1]:
            return
        tile = loaded[i][0]
        old = held.get(tile % slots)
        if old is not None and read_at.get(old, barrier) >= barrier:
            bad.append((old, tile))
        held[tile % slots] = tile
    for i in range(stages):
        load(i)
    for i, (tile, k) in enumerate(loaded):
        barrier += 1
        load(i + stages)
        if k == nk - 1:
            if held[tile % slots] != tile and (tile, held[tile % slots]) not in bad:
                bad.append((tile, held[tile % slots]))
            read_at[tile] = barrier
    return bad


@pytest.mark.parametrize("nk", [1, 2, 3, 10])
def test_no_slot_is_loaded_before_it_was_read(nk):
    stages, slots = _constants()
    assert not _overwritten(12, nk, stages, slots)


def test_two_slots_do_not_hold_tiles_of_one_k_tile():
    """What three slots are for: with two, every tile of one k tile has its slot
    loaded by the tile two further; of more k tiles none."""
    assert len(_overwritten(12, 1, 2, 2)) == 10
    for nk in (2, 3, 10):
        assert not _overwritten(12, nk, 2, 2)


def mm_tile(index: int, grid_m: int, grid_n: int, group_m: int) -> tuple[int, int]:
    """(tile in m, tile in n) of a block's tile, as the kernels' mm_tile."""
    tiles = grid_m * grid_n
    xcd, per, rem = index & 7, tiles >> 3, tiles & 7
    t = xcd * per + min(xcd, rem) + (index >> 3)
    in_group = group_m * grid_n
    first = t // in_group * group_m
    size = min(group_m, grid_m - first)
    i = t % in_group
    return first + i % size, i // size


def row_tiles_change(rows: int, words: int, cus: int = 256) -> int:
    """Tiles of rows x words in 256 x 256 whose block has other rows two tiles on."""
    gm, gn = (words + 255) // 256, (rows + 255) // 256
    tiles = gm * gn
    blocks = min(tiles, cus)
    return sum(mm_tile(i, gm, gn, 4)[1] != mm_tile(i + 2 * blocks, gm, gn, 4)[1]
               for i in range(max(0, tiles - 2 * blocks)))


def test_order_of_tiles():
    for gm, gn in ((1, 1), (3, 5), (64, 12), (197, 3), (257, 8)):
        at = [mm_tile(i, gm, gn, 4) for i in range(gm * gn)]
        assert len(set(at)) == gm * gn
        assert all(0 <= m < gm and 0 <= n < gn for m, n in at)


@pytest.mark.parametrize("rows,words", [(3000, 32768), (700, 50257), (768, 131072),
                                        (2560, 16384), (6000, 20000)])
def test_sizes_of_narrow_heads_meet_other_rows(rows, words):
    """The sizes that the narrow heads' GPU tests take (one k tile, several tiles to a
    block) come to other rows two tiles on: there an overwritten slot changes results.
    2048 rows never do."""
    assert row_tiles_change(rows, words) > 50
    assert row_tiles_change(2048, 65536) == 0
