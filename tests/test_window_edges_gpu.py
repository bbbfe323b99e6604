"""The windowed tree attention: positions that int32 does not hold, and row offsets at its ends."""
from __future__ import annotations

import pytest
import torch

from jetspec_amd import _lib, read_and_clear_status
from test_window_attention_gpu import DEV, attend, trees
from window_helpers import Batch, chain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("position, nearest", [
    (2 ** 33 + 61, 62), (-2 ** 33 + 61, 60), (2 ** 31, 62), (2 ** 32, 62), (2 ** 32 - 1, 62), (-2 ** 31 - 1, 60), (-2 ** 63, 60),
    (2 ** 63 - 1, 62), (-1, 60), (2 ** 31 - 1, 62), (-2 ** 31, 60),
])
def test_int64_positions_outside_are_the_nearer_end(position, nearest):
    # Node 2 of a request over 60 keys.  A window of 2 tells 60, 61 and 62 apart, as the row's position and as the key's.
    b = Batch([50, 60, 70], [chain(5)] * 3, window=2, sinks=0, seed=7)
    p = b.positions.clone()
    p[7] = position
    read_and_clear_status(DEV)
    got = attend(b, positions=p)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_POSITION
    p[7] = nearest
    assert torch.equal(got, attend(b, positions=p))
    assert read_and_clear_status(DEV) == 0
    p[7] = 122 - nearest    # the other end, which would show
    assert not torch.equal(got, attend(b, positions=p))


def test_offsets_of_rows_at_the_ends_of_int32():
    # A request's rows begin past the batch and end at int32's lowest: left out, whatever the difference wraps to.
    def fresh():
        read_and_clear_status(DEV)
        return Batch([50, 60, 70], trees([5, 5, 5]), window=30, seed=7)

    good = attend(fresh())
    for first, last in ((2 ** 30, -2 ** 31), (2 ** 31 - 1, -2 ** 31), (2 ** 31 - 1, 2 ** 31 - 1), (16, -2 ** 31 + 4), (5, -2 ** 31)):
        b = fresh()
        b.meta.cu_seqlens_q[1:3] = torch.tensor([first, last], dtype=torch.int32)
        out = torch.full_like(b.q, 9.0)
        attend(b, out=out)
        assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
        if first == 5:
            assert torch.equal(out[:5], good[:5])
        assert (out[0 if first != 5 else 5:] == 9.0).all(), (first, last)
    b = fresh()
    b.meta.node_counts[1] = 2 ** 31 - 1
    out = torch.full_like(b.q, 9.0)
    attend(b, out=out)
    assert read_and_clear_status(DEV) == _lib.TV_STATUS_BAD_REQUEST
    assert torch.equal(out[:5], good[:5]) and torch.equal(out[10:], good[10:]) and (out[5:10] == 9.0).all()
