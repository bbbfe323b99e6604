"""Pages, slots and requests that do not hold, in every form of the e4m3 tree attention, against 64 bits.

The forms differ in how a missing page is marked: by one staging buffer or by two, a page at a time or key by
key, in a workgroup's first step or in a later one.  Node counts at 4 query heads a KV head choose the row
blocks: 4 -> 32 rows, 16 -> 64, 40 -> 128, 90 -> 256 (head size 256: 128).  The tolerance is Batch.check's.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from jetspec_amd import _lib, read_and_clear_status
from test_e4m3_attention_gpu import BF16, DEV, F32, Batch, trees

pytestmark = pytest.mark.gpu

SIZES = [4, 16, 40, 90]


def drop_pages(batch, request, pages, page):
    """Takes the keys of a request's pages out of what `check` compares with."""
    prefix = batch.prefixes[request]
    gone = np.concatenate([np.arange(p * page, min((p + 1) * page, prefix)) for p in pages])
    batch.keys[request] = np.delete(batch.keys[request], gone)
    batch.prefixes[request] -= gone.size


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dim, page", [(64, 16), (64, 128), (128, 16), (128, 128), (128, 256), (256, 16), (256, 64)])
def test_missing_pages_of_every_row_block(dim, page, size):
    """A share of one step here, so each missing page is in the first step of its workgroup."""
    batch = Batch([5 * page + 5, 3 * page, 90], trees([size] * 3), dim=dim, page=page)
    clean = batch.run(F32)
    for pages, value in (([0], -1), ([0, 1], 10 ** 6), ([3], batch.k.shape[0]), ([5], 2 ** 31 - 1)):
        held = batch.meta.block_tables[0].clone(), batch.keys[0], batch.prefixes[0]
        batch.meta.block_tables[0, pages] = value
        got = batch.run(F32)
        assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_PAGE
        assert torch.equal(got[size:], clean[size:])
        drop_pages(batch, 0, pages, page)
        batch.check(got)
        batch.meta.block_tables[0], batch.keys[0], batch.prefixes[0] = held
    assert torch.equal(batch.run(F32), clean) and read_and_clear_status(DEV) == 0


@pytest.mark.parametrize("dim, page, size", [(64, 128, 90), (64, 16, 90), (128, 128, 90), (128, 16, 90), (128, 128, 40),
                                             (256, 64, 90)])
def test_missing_pages_within_a_share(dim, page, size):
    """More steps than workgroups, so a workgroup runs several: both buffers are marked in turn."""
    batch = Batch([6001, 4000, 4096], trees([size] * 3), dim=dim, page=page, kv_heads=8)
    steps = 3 * 8 * (-(-4 * size // 256)) * (4000 // 128)
    assert steps > 512
    rng = np.random.default_rng(0)
    lost = sorted(rng.choice(4000 // page, size=max(3, 1000 // page), replace=False).tolist())
    for r in (0, 1):
        batch.meta.block_tables[r, lost] = -1
        drop_pages(batch, r, lost, page)
    got = batch.check(BF16)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_PAGE
    for _ in range(3):
        assert torch.equal(batch.run(), got)
    read_and_clear_status(DEV)


POOL_END = "one past the pool"


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dim, page", [(64, 16), (128, 16), (128, 128), (256, 48)])
@pytest.mark.parametrize("bad", [-3, -2 ** 31, -2 ** 40, POOL_END, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 62])
def test_tree_slots_outside_the_pool(bad, dim, page, size):
    """The node is skipped as a key: as if its bias hid it from every row.  Rows that never saw it keep their bits."""
    batch = Batch([40, 90], trees([size, size], seed=size), dim=dim, page=page)
    clean = batch.run(F32)
    node, at = 1, size + 1
    if bad == POOL_END:
        bad = batch.k.shape[0] * page
    elif bad == 2 ** 32 + 1:
        bad = 2 ** 32 + int(batch.meta.tree_slots[at])   # the low half is a slot of the pool
    held = int(batch.meta.tree_slots[at])
    batch.meta.tree_slots[at] = bad
    got = batch.run(F32)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_PAGE
    first = int(batch.meta.qq_bias_offsets[1])
    column = batch.meta.qq_bias[first:first + size * size].view(size, size)[:, node]
    blind = torch.cat([torch.ones(size, dtype=torch.bool, device=DEV), column == -torch.inf])
    assert bool(blind[size]) and not bool(blind[at])
    assert torch.equal(got[blind], clean[blind])
    batch.meta.tree_slots[at] = held
    column.fill_(-torch.inf)
    batch.check(got)
    assert read_and_clear_status(DEV) == 0


@pytest.mark.parametrize("kv_heads, groups, size", [(1, 4, 3), (1, 4, 14), (1, 4, 40), (1, 4, 80), (2, 3, 25)])
@pytest.mark.parametrize("dim, page", [(64, 16), (128, 128), (256, 16)])
def test_more_requests_than_lanes(dim, page, kv_heads, groups, size):
    """Above 64 requests a workgroup's threads search in turn: every row block, with requests that have no nodes,
    lie outside the batch or miss a page."""
    rng = np.random.default_rng(size)
    n = 97
    sizes = rng.integers(max(1, size - 2), size + 3, n)
    batch = Batch([int(x) for x in rng.integers(0, 700, n)], trees(sizes, seed=size), dim=dim, kv_heads=kv_heads,
                  groups=groups, page=page)
    clean = batch.check(F32, requests=range(0, n, 4))
    assert read_and_clear_status(DEV) == 0
    none, outside, missing = {0, 30, 31, 32, 96}, {1, 64, 65}, next(r for r in range(70, n) if batch.prefixes[r] > page)
    for r in none:
        batch.meta.node_counts[r] = 0
    batch.meta.prefix_lens[1] = 10 ** 6
    batch.meta.qq_bias_offsets[64] = -1
    batch.meta.node_counts[65] = 10 ** 6
    batch.meta.block_tables[missing, 1] = -1
    got = batch.run(F32)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST | _lib.TV_STATUS_BAD_PAGE
    batch.meta.qq_bias_offsets[64] = batch.meta.qq_bias_offsets[63] + int(sizes[63]) ** 2
    drop_pages(batch, missing, [1], page)
    kept = [r for r in range(n) if r not in none | outside]
    batch.check(got, requests=[missing, *kept[::5], kept[-1]])
    # The others' work is cut elsewhere now, so a few bits may differ: both are checked against 64 bits.
    assert all(bool(got[batch.meta.request_slice(r)].isfinite().all()) for r in kept)
