"""The e4m3 attention over metadata that is made once and then follows device-built tables and maps, copied into its
fields in place: no host list of the step's own."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from jetspec_amd import (PackedTreeMetadata, build_block_tables, packed_slot_maps, packed_tree_attention_e4m3,
                         read_and_clear_status, workloads)
from test_e4m3_attention_gpu import DEV, F32, Batch, trees

pytestmark = pytest.mark.gpu


def ints(values, kind=torch.int32):
    return torch.tensor(values, dtype=kind, device=DEV)


@pytest.mark.parametrize("captured", [False, True])
def test_fields_follow_the_operators(captured):
    page, sizes, width = 16, [5, 1, 9], 40
    parents = trees(sizes)
    batch = Batch([300, 40, 0], parents, page=page)
    blocks = batch.k.shape[0]
    masks = [torch.as_tensor(workloads.ancestor_mask(t), device=DEV) for t in parents]
    # Made for empty contexts on pages of no matter; as wide as any step's tables.
    spare = list(range(4 * blocks, 4 * blocks + width))
    meta = PackedTreeMetadata.build([width * page, 0, 0], [spare, [], []],
                                    [torch.arange(n, device=DEV) + 64 * i for i, n in enumerate(sizes)], masks, page)
    assert meta.block_tables.shape == (3, width)
    lengths, nodes = ints([0, 0, 0]), ints(sizes)
    arena, free, live = ints([0, 1]), ints(list(range(2, blocks))), ints([blocks - 2])

    def step():
        tables, _, _ = build_block_tables(lengths, free, page, width, free_count=live)
        cu, _, _, _, slots = packed_slot_maps(lengths, nodes, sum(sizes), page, blocks, arena_pages=arena)
        for name, value in (("prefix_lens", lengths), ("block_tables", tables), ("cu_seqlens_q", cu), ("tree_slots", slots)):
            getattr(meta, name).copy_(value)
        return packed_tree_attention_e4m3(batch.q, batch.k, batch.v, batch.ks, batch.vs, meta, batch.scale, 4,
                                          output_dtype=F32)
    for t in (batch.k, batch.v):   # every slot readable
        t.view(torch.uint8)[t.view(torch.uint8) & 127 == 127] = 0x30
    for t in (batch.ks, batch.vs):
        t.nan_to_num_(nan=0.01)
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = step()
    for now in ([200, 40, 0], [0, 0, 0], [17, 160, 33], [1, 16, 255]):
        lengths.copy_(ints(now))
        if captured:
            graph.replay()
            got = result
        else:
            got = step()
        # The same step with metadata built from host lists.
        tables, counts, _ = build_block_tables(lengths, free, page, width)
        _, _, _, _, slots = packed_slot_maps(lengths, nodes, sum(sizes), page, blocks, arena_pages=arena)
        built = PackedTreeMetadata.build(now, [row[:n] for row, n in zip(tables.tolist(), counts.tolist())],
                                         list(torch.split(slots, sizes)), masks, page)
        wide = dataclasses.replace(built, block_tables=tables)
        expect = packed_tree_attention_e4m3(batch.q, batch.k, batch.v, batch.ks, batch.vs, wide, batch.scale, 4,
                                            output_dtype=F32)
        assert torch.equal(got, expect), now
    assert read_and_clear_status(DEV) == 0
