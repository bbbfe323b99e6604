"""Queries of the e4m3 tree attention wherever a tensor of them can begin."""
from __future__ import annotations

import pytest
import torch

from jetspec_amd import read_and_clear_status
from test_e4m3_attention_gpu import BF16, DEV, F16, Batch, trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_dense_queries_off_16_bytes(dim, dtype):
    """A dense tensor that starts inside a buffer is read from a copy, as a strided one is."""
    batch = Batch([70, 0], trees([5, 9]), dim=dim, dtype=dtype)
    q, expect = batch.q, batch.run()
    for shift in (1, 3, 4, 8):
        batch.q = torch.zeros(q.numel() + shift, dtype=dtype, device=DEV)[shift:].view(q.shape)
        batch.q.copy_(q)
        assert batch.q.is_contiguous()
        assert torch.equal(batch.run(), expect)
    assert read_and_clear_status(DEV) == 0
