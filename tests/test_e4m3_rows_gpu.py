"""A row's result in the e4m3 tree attention does not depend on the other rows of its batch: bit for bit."""
from __future__ import annotations

import pytest
import torch

from jetspec_amd import read_and_clear_status
from test_e4m3_attention_gpu import BF16, DEV, F16, F32, Batch, trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, out", [(BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)])
@pytest.mark.parametrize("size", [4, 16, 40, 90])
@pytest.mark.parametrize("dim, page", [(64, 16), (128, 128), (256, 16)])
def test_other_rows_change_no_bit(dim, page, size, dtype, out):
    """Rows whose scores keep growing raise their reference tile after tile; the rows beside them do not."""
    batch = Batch([1500, 700], trees([size, size]), dim=dim, page=page, dtype=dtype)
    before = batch.run(out)
    loud = torch.zeros(batch.q.shape[:2], dtype=torch.bool, device=DEV)
    loud[::3, 1] = loud[1::2, 6] = loud[2, :] = True
    batch.q[loud] *= 40
    got = batch.run(out)
    assert not bool(torch.eq(got[loud], before[loud]).all(-1).any())
    assert torch.equal(got[~loud], before[~loud])
    assert read_and_clear_status(DEV) == 0
