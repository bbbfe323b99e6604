"""The windowed tree attention: positions that int32 does not hold."""
from __future__ import annotations

import pytest
import torch

from jetspec_amd import _lib, read_and_clear_status
from test_window_attention_gpu import DEV, attend
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
