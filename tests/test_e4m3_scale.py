"""Scales whose product with log2(e), which the kernel multiplies by, passes fp32 (CPU: nothing is launched)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from jetspec_amd import PackedTreeMetadata, _lib, packed_tree_attention_e4m3


def call(scale):
    meta = PackedTreeMetadata.build([5], [[0]], [torch.arange(16, 19)], [torch.tril(torch.ones((3, 3), dtype=torch.bool))], 16)
    pool, scales = torch.zeros((2, 16, 2, 64)).to(torch.float8_e4m3fn), torch.zeros((2, 16, 2))
    return packed_tree_attention_e4m3(torch.zeros((3, 8, 64), dtype=torch.bfloat16), pool, pool, scales, scales, meta, scale, 4)


def entry(scale):
    a = _lib.TreeAttentionE4m3Args()
    a.num_requests, a.total_queries, a.num_q_heads, a.num_kv_heads, a.head_dim = 1, 3, 8, 2, 64
    a.num_blocks, a.block_size, a.block_table_width, a.compute_units, a.scale = 2, 16, 1, 256, scale
    return _lib.library().tv_tree_attention_e4m3_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("scale", [2.4e38, 2.5e38, 3e38, -2.4e38, -3e38])
def test_scales_that_leave_fp32_are_refused(scale):
    with np.errstate(over="ignore"):
        assert np.isinf(np.float32(scale) * np.float32(np.log2(np.e)))
    with pytest.raises(ValueError, match="scale must be finite"):
        call(scale)
    assert entry(scale) == _lib.TV_ERR_INVALID


@pytest.mark.parametrize("scale", [2.3e38, -2.3e38, 1.0, 0.0, 1e-44])
def test_scales_that_fit_are_not(scale):
    assert np.isfinite(np.float32(scale) * np.float32(np.log2(np.e)))
    with pytest.raises(ValueError, match="requires GPU tensors"):   # the check after the scale's
        call(scale)
    assert entry(scale) > 0
