"""Refusals of the windowed tree attention (CPU: nothing is launched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from jetspec_amd import PackedTreeMetadata, _lib, packed_window_attention


def operands(dim=64, dtype=torch.bfloat16):
    masks = [torch.tril(torch.ones((n, n), dtype=torch.bool)) for n in (3, 1)]
    meta = PackedTreeMetadata.build([5, 0], [[0], []], [torch.arange(16, 19), torch.tensor([20])], masks, 16)
    pool = torch.zeros((2, 16, 2, dim), dtype=dtype)
    return dict(q=torch.zeros((4, 8, dim), dtype=dtype), k_pool=pool, v_pool=pool.clone(), metadata=meta,
                positions=torch.tensor([5, 6, 7, 0]), scale=0.1, num_queries_per_kv=4, window=8, sinks=1)


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros((5, 8, 64), dtype=torch.bfloat16)), "do not match the metadata"),
    (dict(q=torch.zeros((4, 8, 64))), "BF16 or FP16"),
    (dict(q=torch.zeros((4, 64, 8), dtype=torch.bfloat16).transpose(1, 2)), "head geometry"),
    (dict(q=torch.zeros((4, 8, 96), dtype=torch.bfloat16)), "head geometry"),
    (dict(k_pool=torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16)), "page geometry"),
    (dict(v_pool=torch.zeros((2, 16, 2, 64), dtype=torch.float16)), "share dtype"),
    (dict(num_queries_per_kv=2), "head grouping"),
    (dict(num_queries_per_kv=True), "head grouping"),
    (dict(window=0), "window must be"),
    (dict(window=2 ** 31), "window must be"),
    (dict(window=1.5), "window must be"),
    (dict(window=True), "window must be"),
    (dict(sinks=-1), "sinks must be"),
    (dict(sinks=2 ** 31), "sinks must be"),
    (dict(scale=1e39), "scale must be finite"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(output_dtype=torch.float16), "output dtype"),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), "positions must be"),
    (dict(positions=torch.zeros(4)), "positions must be"),
    (dict(out=torch.zeros((4, 8, 64))), "out must be"),
    (dict(out=torch.zeros((4, 64, 8), dtype=torch.bfloat16).transpose(1, 2)), "out must be"),
    ({}, "requires GPU tensors"),
])
def test_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        packed_window_attention(**(operands() | change))


def test_refuses_outputs_that_overlap():
    given = operands()
    pool = given["k_pool"].view(-1)
    for out in (given["q"], given["q"][:1].expand(4, 8, 64), pool[:2048].view(4, 8, 64)):
        with pytest.raises(ValueError, match="out must"):
            packed_window_attention(**given, out=out)


@pytest.mark.parametrize("dim", [4, 20, 264, 512])
def test_refuses_head_sizes(dim):
    with pytest.raises(ValueError, match="multiples of 8 up to 256"):
        packed_window_attention(**operands(dim))


def block(**over):
    a = _lib.WindowAttentionArgs()
    for name, kind in a._fields_:
        if kind is ctypes.c_void_p:
            setattr(a, name, 0x10000)
    a.q_stride_row, a.q_stride_head, a.out_stride_row, a.out_stride_head = 512, 64, 512, 64
    a.k_stride[:] = a.v_stride[:] = [2048, 128, 64, 1]
    a.in_dtype = a.out_dtype = _lib.TV_BF16
    a.num_blocks, a.block_size, a.block_table_stride, a.block_table_width, a.qq_bias_elems = 8, 16, 4, 4, 16
    a.num_requests, a.total_queries, a.num_q_heads, a.num_kv_heads, a.head_dim = 1, 4, 8, 2, 64
    a.scale, a.window, a.sinks, a.compute_units = 0.1, 8, 0, 256
    for name, value in over.items():
        setattr(a, name, value)
    return a


def test_entry_rejects_bad_arguments_without_a_device():
    lib = _lib.library()
    assert lib.tv_window_attention(None, None, 0, None) == _lib.TV_ERR_INVALID
    assert lib.tv_window_attention_workspace_bytes(None) == _lib.TV_ERR_INVALID
    assert lib.tv_sizeof_window_attention_args() == ctypes.sizeof(_lib.WindowAttentionArgs)
    cases = [
        (dict(num_q_heads=7), _lib.TV_ERR_INVALID, b"query heads over"),
        (dict(head_dim=60), _lib.TV_ERR_UNSUPPORTED, b"head_dim 60"),
        (dict(head_dim=264), _lib.TV_ERR_UNSUPPORTED, b"head_dim 264"),
        (dict(in_dtype=_lib.TV_F32), _lib.TV_ERR_UNSUPPORTED, b"operands"),
        (dict(out_dtype=_lib.TV_F16), _lib.TV_ERR_UNSUPPORTED, b"output"),
        (dict(scale=float("inf")), _lib.TV_ERR_INVALID, b"finite"),
        (dict(window=0), _lib.TV_ERR_INVALID, b"window 0"),
        (dict(sinks=-1), _lib.TV_ERR_INVALID, b"sinks -1"),
        (dict(block_size=0), _lib.TV_ERR_INVALID, b"pool"),
        (dict(num_blocks=2 ** 31, block_size=1), _lib.TV_ERR_UNSUPPORTED, b"2^31 slots"),
        (dict(total_queries=2 ** 30), _lib.TV_ERR_UNSUPPORTED, b"2^31 query rows"),
        (dict(num_requests=-1), _lib.TV_ERR_INVALID, b"negative batch"),
        (dict(positions=None), _lib.TV_ERR_INVALID, b"null pointer"),
        (dict(q=0x10008), _lib.TV_ERR_UNSUPPORTED, b"16 bytes"),
        (dict(out_stride_row=516), _lib.TV_ERR_UNSUPPORTED, b"16 bytes"),
    ]
    for over, code, message in cases:
        assert lib.tv_window_attention(ctypes.byref(block(**over)), 0x10000, 1 << 40, None) == code, over
        assert message in lib.tv_last_error(), (over, lib.tv_last_error())
    # One short prefix over idle compute units is cut, and needs its workspace.
    need = lib.tv_window_attention_workspace_bytes(ctypes.byref(block(block_table_width=1024, window=4096)))
    assert need > 0
    assert lib.tv_window_attention(ctypes.byref(block(block_table_width=1024, window=4096)), 0x10000, need - 1, None) \
        == _lib.TV_ERR_CAPACITY
    assert lib.tv_window_attention(ctypes.byref(block(block_table_width=1024, window=4096)), None, need, None) \
        == _lib.TV_ERR_INVALID
    assert lib.tv_window_attention(ctypes.byref(block(total_queries=0)), None, 0, None) == _lib.TV_OK
    assert lib.tv_window_attention_workspace_bytes(ctypes.byref(block(num_requests=0))) == 0
