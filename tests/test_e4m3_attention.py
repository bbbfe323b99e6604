"""Refusals of the e4m3 tree attention (CPU: nothing is launched)."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch

from jetspec_amd import PackedTreeMetadata, _lib, packed_tree_attention_e4m3

E4M3 = torch.float8_e4m3fn


def operands(dim=64, dtype=torch.bfloat16):
    masks = [torch.tril(torch.ones((n, n), dtype=torch.bool)) for n in (3, 1)]
    meta = PackedTreeMetadata.build([5, 0], [[0], []], [torch.arange(16, 19), torch.tensor([20])], masks, 16)
    pool = torch.zeros((2, 16, 2, dim)).to(E4M3)
    scales = torch.zeros((2, 16, 2))
    return dict(q=torch.zeros((4, 8, dim), dtype=dtype), k_pool=pool, v_pool=pool.clone(), k_scale=scales,
                v_scale=scales.clone(), metadata=meta, scale=0.1, num_queries_per_kv=4)


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros((5, 8, 64), dtype=torch.bfloat16)), "do not match the metadata"),
    (dict(q=torch.zeros((4, 8, 64))), "BF16 or FP16"),
    (dict(q=torch.zeros((4, 64, 8), dtype=torch.bfloat16).transpose(1, 2)), "head geometry"),
    (dict(q=torch.zeros((4, 8, 96), dtype=torch.bfloat16)), "head geometry"),
    (dict(k_pool=torch.zeros((2, 8, 2, 64)).to(E4M3)), "page geometry"),
    (dict(k_pool=torch.zeros((2, 16, 2, 64))), "float8_e4m3fn pools"),
    (dict(v_scale=torch.zeros((2, 16, 1))), "v_scale must be"),
    (dict(k_scale=torch.zeros((2, 16, 2), dtype=torch.float64)), "k_scale must be"),
    (dict(num_queries_per_kv=2), "head grouping"),
    (dict(num_queries_per_kv=True), "head grouping"),
    (dict(num_queries_per_kv=4.0), "head grouping"),
    (dict(output_dtype=torch.float16), "output dtype"),
    (dict(scale=1e39), "scale must be finite"),
    (dict(scale=float("nan")), "scale must be finite"),
    ({}, "requires GPU tensors"),
])
def test_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        packed_tree_attention_e4m3(**(operands() | change))


@pytest.mark.parametrize("dim", [32, 96, 192, 512])
def test_refuses_head_sizes(dim):
    with pytest.raises(ValueError, match="head sizes 64, 128 and 256"):
        packed_tree_attention_e4m3(**operands(dim))


def test_entry_rejects_bad_arguments_without_a_device():
    lib = _lib.library()
    assert lib.tv_tree_attention_e4m3(None, None, 0, None) == _lib.TV_ERR_INVALID
    assert lib.tv_tree_attention_e4m3_workspace_bytes(None) == _lib.TV_ERR_INVALID
    assert lib.tv_sizeof_tree_attention_e4m3_args() == ctypes.sizeof(_lib.TreeAttentionE4m3Args)

    def block(**over):
        a = _lib.TreeAttentionE4m3Args()
        for name, kind in a._fields_:
            if kind is ctypes.c_void_p:
                setattr(a, name, 0x10000)
        a.q_stride_row = a.out_stride_row = 1024
        a.q_stride_head = a.out_stride_head = 128
        a.k_stride[:] = a.v_stride[:] = (4096, 256, 128, 1)
        a.k_scale_stride[:] = a.v_scale_stride[:] = (32, 2, 1)
        a.num_blocks, a.block_size, a.block_table_stride, a.block_table_width, a.qq_bias_elems = 4, 16, 2, 2, 9
        a.num_requests, a.total_queries, a.num_q_heads, a.num_kv_heads, a.head_dim = 1, 3, 8, 2, 128
        a.scale, a.compute_units = 0.1, 256
        for name, value in over.items():
            setattr(a, name, value)
        return a

    def launch(workspace=0x10000, size=1 << 40, **over):
        return lib.tv_tree_attention_e4m3(ctypes.byref(block(**over)), workspace, size, None)
    invalid, unsupported = _lib.TV_ERR_INVALID, _lib.TV_ERR_UNSUPPORTED
    for over, code in ((dict(num_requests=-1), invalid), (dict(total_queries=-1), invalid), (dict(num_q_heads=7), invalid),
                       (dict(num_kv_heads=0), invalid), (dict(head_dim=96), unsupported), (dict(in_dtype=2), unsupported),
                       (dict(out_dtype=1), unsupported), (dict(scale=float("nan")), invalid), (dict(scale=float("inf")), invalid),
                       (dict(num_blocks=0), invalid), (dict(block_size=0), invalid), (dict(block_table_width=-1), invalid),
                       (dict(num_blocks=1 << 28), unsupported), (dict(total_queries=1 << 29), unsupported),
                       (dict(compute_units=0), invalid)):
        assert launch(**over) == code, over
        assert lib.tv_tree_attention_e4m3_workspace_bytes(ctypes.byref(block(**over))) == code, over
    for over in (dict(q=None), dict(k_scale=None), dict(tree_slots=None), dict(qq_bias=None)):
        assert launch(**over) == invalid, over
    for over in (dict(q=0x10008), dict(q_stride_head=4), dict(k_pool=0x10004), dict(out=0x10008), dict(out_stride_row=4)):
        assert launch(**over) == unsupported, over
    assert launch(workspace=None) == invalid and launch(workspace=0x10008) == invalid
    need = lib.tv_tree_attention_e4m3_workspace_bytes(ctypes.byref(block()))
    assert need > 0 and launch(size=need - 1) == _lib.TV_ERR_CAPACITY
    assert launch(num_requests=0) == _lib.TV_OK and launch(total_queries=0) == _lib.TV_OK
    empty = block(num_requests=0)
    assert lib.tv_tree_attention_e4m3_workspace_bytes(ctypes.byref(empty)) == 0


def test_the_workspace_covers_every_shape():
    """Two pieces a workgroup, of a row block's rows, for the rows that an average request has."""
    lib = _lib.library()
    for dim, rows_of in ((64, (32, 64, 128, 256)), (128, (32, 64, 128, 256)), (256, (32, 64, 128, 128))):
        for average, rows in zip((20, 60, 100, 5000), rows_of):
            a = _lib.TreeAttentionE4m3Args()
            a.num_requests, a.total_queries, a.num_q_heads, a.num_kv_heads, a.head_dim = 40, 40 * average, 2, 2, dim
            a.num_blocks, a.block_size, a.block_table_width, a.compute_units, a.scale = 1 << 20, 256, 100, 256, 1.0
            size = lib.tv_tree_attention_e4m3_workspace_bytes(ctypes.byref(a))
            groups, rest = divmod(size, 2 * rows * (4 * dim + 8) + 16)   # and a job of 16 bytes
            assert rest == 0 and groups in (256, 512), (dim, average)


def test_packed_arguments_are_the_structure():
    """The bytes that an entry gets are those of the structure filled field by field."""
    for pack, kind in ((_lib.pack_qk_norm, _lib.QkNormArgs), (_lib.pack_store_e4m3, _lib.StoreE4m3Args),
                       (_lib.pack_tree_attention_e4m3, _lib.TreeAttentionE4m3Args)):
        values = []

        def fill(block):
            for name, field in block._fields_:
                if issubclass(field, ctypes.Structure):
                    fill(getattr(block, name))
                elif issubclass(field, ctypes.Array):
                    for i in range(field._length_):
                        values.append(len(values) + 1)
                        getattr(block, name)[i] = values[-1]
                else:
                    values.append(len(values) + 1)
                    setattr(block, name, values[-1])
        block = kind()
        fill(block)
        assert pack(*values) == bytes(block)
