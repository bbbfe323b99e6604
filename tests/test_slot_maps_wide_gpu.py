"""int64 cache lengths and depths that no int32 holds: reported, never mapped to another position."""
from __future__ import annotations

import pytest
import torch

from jetspec_amd import _lib, packed_slot_maps, read_and_clear_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(*values, kind=torch.int64):
    return torch.tensor(values, dtype=kind, device=DEV)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("far", [2 ** 31, 2 ** 32 + 3, 2 ** 40, 2 ** 63 - 1, -1, -2 ** 31 - 1, -2 ** 32 + 3, -2 ** 63])
def test_cache_lengths(far, paged):
    pages = dict(block_tables=ints(5, 6, 7).view(1, 3).repeat(3, 1)) if paged else dict(arena_pages=ints(5, 6, 7))
    _, request, local, positions, slots = packed_slot_maps(ints(1, far, 2), ints(1, 2, 1), 4, 4, 8, **pages)
    assert request.tolist() == [0, 1, 1, 2] and local.tolist() == [0, 0, 1, 0]
    assert positions.tolist() == [1, 0, 0, 2]
    assert slots.tolist() == ([21, -1, -1, 22] if paged else [20, -1, -1, 23])
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_POSITION


@pytest.mark.parametrize("far", [2 ** 31, 2 ** 32 + 1, 2 ** 63 - 1, -2 ** 31 - 1, -2 ** 32 + 1, -2 ** 63])
def test_depths(far):
    got = packed_slot_maps(ints(10, 0), ints(2, 1), 3, 4, 8, arena_pages=ints(5), depths=ints(0, far, 3))
    assert got[3].tolist() == [10, 0, 3] and got[4].tolist() == [20, -1, 22]
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_POSITION


def test_the_largest_that_int32_holds():
    top = 2 ** 31 - 1
    got = packed_slot_maps(ints(top, 0), ints(2, 1), 3, 4, 8, arena_pages=ints(5), depths=ints(0, 5, top))
    assert got[3].tolist() == [top, top + 5, top] and got[4].tolist() == [20, 21, 22]
    got = packed_slot_maps(ints(9), ints(2), 2, 4, 8, arena_pages=ints(5), depths=ints(-4, -9))
    assert got[3].tolist() == [5, 0] and got[4].tolist() == [20, 21]
    assert read_and_clear_status(DEV) == 0
