"""Block tables and slot maps on the GPU against host loops, entry for entry."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from jetspec_amd import PackedTreeMetadata, _lib, build_block_tables, packed_slot_maps, read_and_clear_status, workloads

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(values, kind=torch.int32):
    return torch.as_tensor(np.asarray(values), dtype=kind, device=DEV)


def tables_by_loop(lengths, free, page, width, held, counts):
    """The definition, request by request."""
    rows, out, at, short = [], [], 0, False
    for length, row, count in zip(lengths, held, counts):
        need = -(-int(length) // page)
        pages = list(row[:count])
        if count < need <= width:
            short = short or at + need - count > len(free)
            if not short:
                pages += list(free[at:at + need - count])
                at += need - count
        out.append(len(pages))
        rows.append(pages + [-1] * (width - len(pages)))
    return np.array(rows).reshape(len(out), width), np.array(out), at


def check_tables(lengths, free, page, width, held=None, counts=None, **more):
    n = len(lengths)
    call = dict(held_tables=ints(held), held_counts=ints(counts)) if held is not None else {}
    tables, got, taken = build_block_tables(ints(lengths), ints(free), page, width, **call, **more)
    expect = tables_by_loop(lengths, free, page, width, held if held is not None else np.zeros((n, 0)),
                            counts if counts is not None else np.zeros(n, dtype=int))
    np.testing.assert_array_equal(tables.cpu().numpy(), expect[0])
    np.testing.assert_array_equal(got.cpu().numpy(), expect[1])
    assert int(taken) == expect[2]


@pytest.mark.parametrize("requests, page, top, width", [
    (1, 16, 1, 1), (1, 256, 70000, 274), (7, 1, 33, 40), (64, 256, 32768, 128), (257, 48, 900, 19),
    (1023, 16, 300, 20), (1500, 16, 2000, 125), (5000, 7, 60, 9),
])
def test_admission_and_growth(requests, page, top, width):
    rng = np.random.default_rng(requests)
    lengths = rng.integers(0, top + 1, size=requests)
    lengths[rng.integers(requests)] = top
    need = -(-lengths // page)
    free = rng.permutation(int(need.sum()) + 5)
    check_tables(lengths, free, page, width)
    counts = np.minimum((need * rng.random(requests)).astype(int) + rng.integers(0, 2, requests), width)
    held = rng.integers(0, 1 << 20, size=(requests, width))
    check_tables(lengths, free, page, width, held, counts)
    # A held table narrower than the new one, as a view of a wider store.
    store = ints(held)
    low = max(1, width // 2)
    counts = np.minimum(counts, low)
    tables, got, _ = build_block_tables(ints(lengths, torch.int64), ints(free), page, width,
                                        held_tables=store[:, :low], held_counts=ints(counts))
    expect = tables_by_loop(lengths, free, page, width, held[:, :low], counts)
    np.testing.assert_array_equal(tables.cpu().numpy(), expect[0])
    np.testing.assert_array_equal(got.cpu().numpy(), expect[1])
    assert read_and_clear_status(DEV) == 0


@pytest.mark.parametrize("requests", [3, 300, 3000])
def test_a_short_list_stops_at_the_first_request_it_cannot_serve(requests):
    rng = np.random.default_rng(requests)
    lengths = rng.integers(0, 200, size=requests)
    need = -(-lengths // 16)
    for have in sorted({0, 1, int(need.sum()) // 2, int(need.sum()) - 1}):
        check_tables(lengths, rng.permutation(have), 16, 13)
        # The same list inside a longer buffer, its length on the device.
        longer = np.concatenate([rng.permutation(have), np.full(100, -7)])
        tables, got, taken = build_block_tables(ints(lengths), ints(longer), 16, 13, free_count=ints([have]))
        expect = tables_by_loop(lengths, longer[:have], 16, 13, np.zeros((requests, 0)), np.zeros(requests, dtype=int))
        np.testing.assert_array_equal(tables.cpu().numpy(), expect[0])
        np.testing.assert_array_equal(got.cpu().numpy(), expect[1])
        assert int(taken) == expect[2]
        short = need.sum() > have
        assert read_and_clear_status(DEV) == (_lib.TV_STATUS_NO_PAGES if short else 0)


def test_a_request_wider_than_the_table_takes_nothing():
    check_tables([10, 1000, 20], np.arange(40), 10, 5)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_NO_PAGES


def test_bad_lengths_and_counts_are_clamped():
    tables, counts, taken = build_block_tables(ints([-5, 20]), ints([3, 4, 5]), 10, 4,
                                               held_tables=ints([[8, 9], [8, 9]]), held_counts=ints([-1, 7]))
    assert tables.tolist() == [[-1] * 4, [8, 9, -1, -1]] and counts.tolist() == [0, 2] and taken.tolist() == [0]
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
    _, counts, taken = build_block_tables(ints([20]), ints([3, 4]), 10, 4, free_count=ints([9]))
    assert counts.tolist() == [2] and taken.tolist() == [2]
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST


def test_values_past_32_bits_do_not_wrap():
    """2^32 + 3 in an int64 input is no 3: too long, too far or no page, as the nearest 32-bit value is."""
    far = torch.tensor([2 ** 32 + 3, 5], device=DEV)
    _, counts, taken = build_block_tables(far, ints([3, 4]), 10, 4)
    assert counts.tolist() == [0, 1] and taken.tolist() == [1]
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_NO_PAGES
    slots = packed_slot_maps(ints([0, 0]), ints([1, 1]), 2, 4, 8, block_tables=far.unsqueeze(1))[4]
    assert slots.tolist() == [-1, 20]
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_SLOT


def test_no_requests():
    tables, counts, taken = build_block_tables(ints([]), ints([1, 2]), 16, 3)
    assert tables.shape == (0, 3) and counts.numel() == 0 and taken.tolist() == [0]


def maps_by_loop(cached, rows, total, page, tables=None, arena=None, depths=None):
    request, local, position, slot, cu = [], [], [], [], [0]
    for r, (c, n) in enumerate(zip(cached, rows)):
        for l in range(int(n)):
            i = len(request)
            request.append(r)
            local.append(l)
            position.append(int(c) + (l if depths is None else int(depths[i])))
            at = i if arena is not None else int(c) + l
            entry = arena[at // page] if arena is not None else tables[r][at // page]
            slot.append(int(entry) * page + at % page)
        cu.append(cu[-1] + int(n))
    pad = total - len(request)
    return cu, request + [-1] * pad, local + [0] * pad, position + [0] * pad, slot + [-1] * pad


@pytest.mark.parametrize("requests, rows, page, pad, arena", [
    (1, 1, 16, 0, False), (1, 700, 48, 13, False), (250, 1, 256, 6, False), (9, 300, 1, 0, True), (33, 64, 256, 0, True),
    (1024, 3, 16, 7, False), (1025, 3, 16, 0, True), (4100, 2, 16, 1, False), (3, 120000, 256, 300, False),
])
def test_maps(requests, rows, page, pad, arena):
    rng = np.random.default_rng(requests + rows)
    cached = rng.integers(0, 1000, size=requests)
    lens = rng.integers(0, rows + 1, size=requests)
    lens[-1] = rows
    total = int(lens.sum()) + pad
    depths = rng.integers(0, 9, size=total) if arena else None
    width = -(-(1000 + rows) // page)
    blocks = 1 << 20
    tables = rng.integers(0, blocks, size=(requests, width))
    pages = rng.permutation(-(-total // page) + 1)
    got = packed_slot_maps(ints(cached), ints(lens), total, page, blocks, block_tables=None if arena else ints(tables),
                           arena_pages=ints(pages) if arena else None, depths=ints(depths) if arena else None)
    expect = maps_by_loop(cached, lens, total, page, tables, pages if arena else None, depths)
    for name, x, y in zip(("cu", "request", "local", "positions", "slots"), got, expect):
        np.testing.assert_array_equal(x.cpu().numpy(), np.asarray(y), err_msg=name)
    assert [t.dtype for t in got] == [torch.int32] * 3 + [torch.int64] * 2
    assert read_and_clear_status(DEV) == 0


def test_maps_of_nothing():
    cu, *rest = packed_slot_maps(ints([]), ints([]), 3, 16, 4, block_tables=torch.empty((0, 2), dtype=torch.int32, device=DEV))
    assert cu.tolist() == [0] and [t.tolist() for t in rest] == [[-1] * 3, [0] * 3, [0] * 3, [-1] * 3]
    cu, *rest = packed_slot_maps(ints([5, 6]), ints([0, 0]), 0, 16, 4, arena_pages=ints([]))
    assert cu.tolist() == [0, 0, 0] and all(t.numel() == 0 for t in rest)


def test_bad_pages_positions_and_lengths():
    tables = ints([[0, 9, -1], [1, 2, 3]])
    got = packed_slot_maps(ints([3, 10]), ints([6, 4]), 10, 4, 4, block_tables=tables)
    # Page 9 lies outside 4 blocks, the third entry is no page, and position 12 is past the second table.
    assert got[4].tolist() == [3, -1, -1, -1, -1, -1, 14, 15, -1, -1]
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_SLOT
    got = packed_slot_maps(ints([-1, 0]), ints([2, 2]), 4, 4, 8, block_tables=tables)
    assert got[4].tolist() == [-1, -1, 4, 5] and min(got[3].tolist()) == 0
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_POSITION
    got = packed_slot_maps(ints([0, 0]), ints([-3, 2]), 2, 4, 8, block_tables=tables)
    assert got[0].tolist() == [0, 0, 2] and got[4].tolist() == [4, 5]
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
    got = packed_slot_maps(ints([0, 0]), ints([2, 5]), 3, 4, 8, block_tables=tables)
    assert got[0].tolist() == [0, 2, 7] and got[1].tolist() == [0, 0, 1] and got[4].tolist() == [0, 1, 4]
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
    got = packed_slot_maps(ints([2 ** 31 - 1]), ints([2]), 2, 4, 8, block_tables=ints([[0]]))
    assert got[4].tolist() == [-1, -1] and got[3].tolist() == [2 ** 31 - 1, 2 ** 31]
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_SLOT


def test_tree_maps_equal_the_packed_metadata():
    """The maps of a tree batch are the fields that the metadata constructor makes on the host."""
    rng = np.random.default_rng(3)
    counts = [16, 1, 40, 64]
    prefixes = [300, 0, 17, 1024]
    trees = [workloads.random_parents(n, 8, rng) for n in counts]
    pages = [list(range(100 * r, 100 * r + -(-p // 32))) for r, p in enumerate(prefixes)]
    arena = [500, 400, 401, 77]
    node = np.arange(sum(counts))
    slots = torch.as_tensor(np.asarray(arena)[node // 32] * 32 + node % 32, device=DEV)
    masks = [torch.as_tensor(workloads.ancestor_mask(t), device=DEV) for t in trees]
    meta = PackedTreeMetadata.build(prefixes, pages, list(torch.split(slots, counts)), masks, 32)
    depths = ints(np.concatenate([workloads.depths_of(t) for t in trees]))
    cu, request, local, positions, got = packed_slot_maps(ints(prefixes), ints(counts), sum(counts), 32, 600,
                                                          arena_pages=ints(arena), depths=depths)
    assert torch.equal(cu, meta.cu_seqlens_q) and torch.equal(request, meta.query_to_request)
    assert torch.equal(local, meta.query_local_row) and torch.equal(got, meta.tree_slots)
    assert torch.equal(positions, ints(prefixes)[request.long()].long() + depths.long())


def test_capture_follows_the_lengths():
    lengths, counts, held = ints([5, 40, 0]), ints([1, 2, 0]), ints([[7, -1, -1], [8, 9, -1], [-1] * 3])
    free, live, rows = ints([20, 21, 22, 23]), ints([4]), ints([1, 2, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        made = build_block_tables(lengths + rows, free, 16, 3, held_tables=held, held_counts=counts, free_count=live)
        return made, packed_slot_maps(lengths, rows, 6, 16, 64, block_tables=made[0])
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        lengths.copy_(ints([5 + 11 * k, 40 - k, 3 * k]))
        rows.copy_(ints([1, 2, k]))
        live.copy_(ints([4 - k]))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        for x, y in zip((*captured[0], *captured[1]), (*eager[0], *eager[1])):
            assert torch.equal(x, y), k
    read_and_clear_status(DEV)
