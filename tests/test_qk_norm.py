"""Refusals of the fused Q/K norm and of the e4m3 append, and the e4m3 oracle itself (CPU)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import e4m3_helpers
from jetspec_amd import _lib, qk_norm_rope_scatter, qk_norm_rope_scatter_prevalidated, store_kvcache_e4m3

E4M3 = torch.float8_e4m3fn


def test_oracle_codes_are_the_type_s_values():
    codes = torch.arange(256, dtype=torch.uint8)
    np.testing.assert_array_equal(e4m3_helpers.VALUES, codes.view(E4M3).double().numpy())
    # Every midpoint, its neighbours and the values themselves round as the type's own conversion does.
    ladder = e4m3_helpers.VALUES[:127]
    middle = ((ladder[1:] + ladder[:-1]) / 2).astype(np.float32)
    x = np.concatenate([ladder.astype(np.float32), middle, np.nextafter(middle, np.float32(0)),
                        np.nextafter(middle, np.float32(1e9))])
    x = np.concatenate([x, -x])
    np.testing.assert_array_equal(e4m3_helpers.encode(x), torch.from_numpy(x).to(E4M3).view(torch.uint8).numpy())


def operands(rows=3, q_heads=4, kv_heads=2, dim=64, e4m3=False, dtype=torch.bfloat16):
    def t(*shape, kind=dtype):
        return torch.zeros(shape, dtype=torch.float32).to(kind)
    pool = E4M3 if e4m3 else dtype
    call = dict(q=t(rows, q_heads, dim), k=t(rows, kv_heads, dim), v=t(rows, kv_heads, dim), q_weight=t(dim), k_weight=t(dim),
                positions=torch.zeros(rows, dtype=torch.int64), cos_sin_cache=t(16, dim, kind=torch.float32),
                k_pool=t(2, 16, kv_heads, dim, kind=pool), v_pool=t(2, 16, kv_heads, dim, kind=pool),
                node_slots=torch.arange(rows))
    if e4m3:
        call |= dict(k_scale=t(2, 16, kv_heads, kind=torch.float32), v_scale=t(2, 16, kv_heads, kind=torch.float32))
    return call


def z(*shape, kind=torch.bfloat16):
    return torch.zeros(shape, dtype=torch.float32).to(kind)


@pytest.mark.parametrize("e4m3, change, message", [
    (False, dict(q=z(3, 256)), "rows,heads,dim"),
    (False, dict(v=z(3, 1, 64)), "equal K/V geometry"),
    (False, dict(q=z(3, 5, 64)), "head geometry"),
    (False, dict(q=z(2, 4, 64)), "head geometry"),
    (False, dict(q=z(3, 4, 64, kind=torch.float16)), "share one of"),
    (False, dict(positions=torch.zeros(3)), "integer .rows. vectors"),
    (False, dict(node_slots=torch.zeros(2, dtype=torch.int64)), "integer .rows. vectors"),
    (False, dict(cos_sin_cache=z(16, 32)), "cos/sin cache"),
    (False, dict(cos_sin_cache=z(16, 64, kind=torch.float16)), "cos/sin cache"),
    (False, dict(q_weight=z(32)), "norm weights"),
    (False, dict(k_weight=z(64, kind=torch.float32)), "norm weights"),
    (False, dict(q_weight=z(128)[::2]), "norm weights"),
    (False, dict(k_pool=z(2, 16, 2, 64, kind=torch.float32)), "KV pools must match"),
    (False, dict(k_pool=z(2, 16, 3, 64)), "KV pools must match"),
    (False, dict(k_scale=z(2, 16, 2, kind=torch.float32)), "scales belong"),
    (True, dict(k_scale=None), "k_scale must be"),
    (True, dict(v_scale=z(2, 16, 2)), "v_scale must be"),
    (True, dict(v_scale=z(2, 16, 1, kind=torch.float32)), "v_scale must be"),
    (True, dict(v_pool=z(2, 16, 2, 64)), "KV pools must match"),
    (True, dict(v_scale=z(2, 16, 1, kind=torch.float32).expand(2, 16, 2)), "positive strides"),
    (False, dict(eps=float("nan")), "eps must be"),
    (False, dict(eps=-1.0), "eps must be"),
    (False, dict(eps=1e39), "eps must be"),
    (False, {}, "requires GPU tensors"),
    (True, {}, "requires GPU tensors"),
])
def test_qk_norm_refuses(e4m3, change, message):
    call = operands(e4m3=e4m3) | change
    with pytest.raises(ValueError, match=message):
        qk_norm_rope_scatter(**call)
    with pytest.raises(ValueError, match=message):
        qk_norm_rope_scatter_prevalidated(**call, out=torch.zeros_like(call["q"]))


@pytest.mark.parametrize("dim", [1, 63, 258])
def test_qk_norm_refuses_head_sizes(dim):
    with pytest.raises(ValueError, match="head geometry"):
        qk_norm_rope_scatter(**operands(dim=dim))


def test_qk_norm_refuses_another_output():
    with pytest.raises(ValueError, match="output must match"):
        qk_norm_rope_scatter(**operands(), out=z(3, 4, 32))
    with pytest.raises(ValueError, match="output must match"):
        qk_norm_rope_scatter_prevalidated(**operands(), out=z(3, 4, 64, kind=torch.float32))


def store_operands():
    return dict(key=z(3, 2, 64), value=z(3, 2, 64), k_cache=z(2, 16, 2, 64, kind=E4M3), v_cache=z(2, 16, 2, 64, kind=E4M3),
                k_scale=z(2, 16, 2, kind=torch.float32), v_scale=z(2, 16, 2, kind=torch.float32),
                slot_mapping=torch.arange(3))


@pytest.mark.parametrize("change, message", [
    (dict(value=z(3, 2, 32)), "one shape and dtype"),
    (dict(key=z(3, 2, 64, kind=torch.float32)), "one shape and dtype"),
    (dict(key=z(3, 2, 63), value=z(3, 2, 63)), "even head sizes"),
    (dict(k_cache=z(2, 16, 2, 64)), "caches must be"),
    (dict(v_cache=z(2, 8, 2, 64, kind=E4M3)), "caches must be"),
    (dict(k_scale=z(2, 16, 2)), "k_scale must be"),
    (dict(slot_mapping=torch.arange(2)), "slot_mapping"),
    (dict(slot_mapping=torch.zeros(3)), "slot_mapping"),
    ({}, "requires GPU tensors"),
])
def test_store_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        store_kvcache_e4m3(**(store_operands() | change))


def test_entries_reject_bad_arguments_without_a_device():
    lib = _lib.library()
    assert lib.tv_qk_norm_rope_scatter(None, None) == _lib.TV_ERR_INVALID
    assert lib.tv_store_kvcache_e4m3(None, None) == _lib.TV_ERR_INVALID
    assert lib.tv_sizeof_qk_norm_args() == ctypes.sizeof(_lib.QkNormArgs)
    assert lib.tv_sizeof_store_e4m3_args() == ctypes.sizeof(_lib.StoreE4m3Args)

    def norm(**over):
        a = _lib.QkNormArgs()
        r = a.rope
        r.q = r.k = r.v = r.positions = r.cache = r.k_pool = r.v_pool = r.node_slots = r.out = 0x10000
        a.q_weight = a.k_weight = 0x10000
        r.q_stride[:], r.k_stride[:], r.v_stride[:], r.out_stride[:] = (256, 64, 1), (128, 64, 1), (128, 64, 1), (256, 64, 1)
        r.k_pool_stride[:] = r.v_pool_stride[:] = (2048, 128, 64, 1)
        r.positions_stride = r.slots_stride = r.cache_stride_elem = 1
        r.cache_stride_row, r.cache_rows, r.pool_pages, r.page_size = 64, 16, 2, 16
        r.rows, r.q_heads, r.kv_heads, r.head_dim = 3, 4, 2, 64
        for name, value in over.items():
            setattr(a if hasattr(a, name) else r, name, value)
        return lib.tv_qk_norm_rope_scatter(ctypes.byref(a), None)
    invalid, unsupported = _lib.TV_ERR_INVALID, _lib.TV_ERR_UNSUPPORTED
    for over, code in ((dict(rows=-1), invalid), (dict(q_heads=5), invalid), (dict(kv_heads=0), invalid),
                       (dict(head_dim=63), invalid), (dict(head_dim=258), invalid), (dict(dtype=3), unsupported),
                       (dict(cache_dtype=1), unsupported), (dict(weight_dtype=1), unsupported), (dict(eps=-1.0), invalid),
                       (dict(eps=float("nan")), invalid), (dict(out=None), invalid), (dict(q_weight=None), invalid),
                       (dict(pool_e4m3=1), invalid), (dict(cache_rows=0), invalid), (dict(page_size=0), invalid),
                       (dict(slots_stride=0), invalid), (dict(rows=1 << 31), unsupported)):
        assert norm(**over) == code, over
    assert norm(rows=0) == _lib.TV_OK

    def store(**over):
        a = _lib.StoreE4m3Args()
        a.key = a.value = a.k_cache = a.v_cache = a.k_scale = a.v_scale = a.slots = 0x10000
        a.key_stride[:] = a.value_stride[:] = (128, 64, 1)
        a.k_cache_stride[:] = a.v_cache_stride[:] = (2048, 128, 64, 1)
        a.k_scale_stride[:] = a.v_scale_stride[:] = (32, 2, 1)
        a.slots_stride, a.pool_pages, a.page_size, a.rows, a.kv_heads, a.head_dim = 1, 2, 16, 3, 2, 64
        for name, value in over.items():
            setattr(a, name, value)
        return lib.tv_store_kvcache_e4m3(ctypes.byref(a), None)
    for over, code in ((dict(rows=-1), invalid), (dict(kv_heads=0), invalid), (dict(head_dim=0), invalid),
                       (dict(dtype=7), unsupported), (dict(key=None), invalid), (dict(v_scale=None), invalid),
                       (dict(pool_pages=0), invalid), (dict(slots_stride=0), invalid), (dict(rows=1 << 31), unsupported)):
        assert store(**over) == code, over
    assert store(rows=0) == _lib.TV_OK


def test_the_launch_only_form_needs_an_output():
    with pytest.raises(ValueError, match="given output"):
        qk_norm_rope_scatter_prevalidated(**operands(), out=None)
