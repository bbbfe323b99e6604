"""Queries of the packed and the single-request attention wherever a dense tensor of them can begin."""
from __future__ import annotations

import pytest
import torch

from jetspec_amd import packed_tree_attention, packed_tree_attention_reference, read_and_clear_status
from test_attention_gpu import reference_fixture
from test_legacy_exact_gpu import SCALE, legacy_call

pytestmark = pytest.mark.gpu


def moved(q, shift):
    copy = torch.zeros(q.numel() + shift, dtype=q.dtype, device=q.device)[shift:].view(q.shape).copy_(q)
    assert copy.is_contiguous() and copy.data_ptr() % 16 == shift * q.element_size() % 16
    return copy


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [1, 4, 8])
def test_dense_queries_off_16_bytes(shift, dtype):
    q, k, v, meta, slots, masks, _ = reference_fixture(dtype=dtype)
    for call in (packed_tree_attention, packed_tree_attention_reference):
        assert torch.equal(call(moved(q, shift), k, v, meta, SCALE, 4), call(q, k, v, meta, SCALE, 4))
    mine = q[meta.request_slice(0)].contiguous()
    request = (k, v, meta.prefix_lengths[0], meta.block_tables_host[0], slots[0], masks[0])
    assert torch.equal(legacy_call(moved(mine, shift), *request), legacy_call(mine, *request))
    assert read_and_clear_status(q.device) == 0
