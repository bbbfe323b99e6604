"""Refusals of the block-table and slot-map operators (CPU: nothing is launched)."""
from __future__ import annotations

import pytest
import torch

from jetspec_amd import _lib, build_block_tables, packed_slot_maps


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.mark.parametrize("change, message", [
    (dict(block_size=0), "positive block size"),
    (dict(width=0), "positive block size"),
    (dict(lengths=torch.zeros(2)), "int32 or int64 vector"),
    (dict(lengths=torch.zeros((1, 2), dtype=torch.int32)), "int32 or int64 vector"),
    (dict(held_tables=torch.zeros((2, 4), dtype=torch.int32)), "come together"),
    (dict(held_counts=ints(0, 0)), "come together"),
    (dict(held_tables=torch.zeros((2, 9), dtype=torch.int32), held_counts=ints(0, 0)), "fit the table width"),
    (dict(held_tables=torch.zeros((2, 4), dtype=torch.int32), held_counts=ints(0)), "match the requests"),
    (dict(held_tables=torch.zeros((3, 4), dtype=torch.int32), held_counts=ints(0, 0)), "held_tables must be"),
    (dict(free_count=ints(1, 2)), "one integer"),
    ({}, "requires GPU tensors"),
])
def test_build_block_tables_refuses(change, message):
    call = dict(lengths=ints(3, 4), free_pages=ints(0, 1, 2), block_size=2, width=8)
    call.update(change)
    with pytest.raises(ValueError, match=message):
        build_block_tables(**call)


@pytest.mark.parametrize("change, message", [
    (dict(total_rows=-1), "row count"),
    (dict(block_size=0), "positive block size"),
    (dict(num_blocks=0), "positive pool size"),
    (dict(block_tables=None), "either block_tables or arena_pages"),
    (dict(arena_pages=ints(0)), "either block_tables or arena_pages"),
    (dict(query_lens=ints(1)), "request count"),
    (dict(query_lens=torch.ones(2)), "int32 or int64 vector"),
    (dict(block_tables=torch.zeros((1, 3), dtype=torch.int32)), "block_tables must be"),
    (dict(depths=ints(0)), "one entry per packed row"),
    ({}, "requires GPU tensors"),
])
def test_packed_slot_maps_refuses(change, message):
    call = dict(cache_lens=ints(3, 4), query_lens=ints(1, 1), total_rows=2, block_size=4, num_blocks=8,
                block_tables=torch.zeros((2, 2), dtype=torch.int32))
    call.update(change)
    with pytest.raises(ValueError, match=message):
        packed_slot_maps(**call)


def test_entries_reject_bad_arguments_without_a_device():
    lib = _lib.library()

    def tables(requests=1, block=16, width=4, capacity=4, held=0, taken=0x1000, free=0x1000):
        return lib.tv_build_block_tables(0x1000, None, 0, held, None, free, None, capacity, requests, block, width, 0x1000,
                                         0x1000, taken, None, None)
    for bad in (dict(requests=-1), dict(block=0), dict(width=0), dict(capacity=-1), dict(held=5), dict(taken=None),
                dict(free=None)):
        assert tables(**bad) == _lib.TV_ERR_INVALID, bad

    def maps(requests=1, rows=1, block=16, blocks=4, paged=0x1000, arena=None, cu=0x1000):
        return lib.tv_packed_slot_maps(0x1000, 0x1000, paged, 4, 4, arena, 4, None, requests, rows, block, blocks, cu,
                                       0x1000, 0x1000, 0x1000, 0x1000, None, None)
    for bad in (dict(requests=-1), dict(rows=-1), dict(rows=1 << 31), dict(block=0), dict(blocks=0), dict(paged=None),
                dict(arena=0x1000), dict(cu=None)):
        assert maps(**bad) == _lib.TV_ERR_INVALID, bad
