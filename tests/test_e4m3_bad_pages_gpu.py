"""Pages and slots outside the pool in every form of the e4m3 tree attention, against 64 bits.

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
