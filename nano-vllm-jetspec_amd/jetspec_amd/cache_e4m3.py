"""An 8-bit K/V cache: e4m3 rows with a scale per slot and head, and the operators on it.

``k_cache`` and ``v_cache`` are float8_e4m3fn [pages, page_size, kv_heads, dim]; ``k_scale`` and
``v_scale`` float32 [pages, page_size, kv_heads].  A row of one head reads as ``code * scale`` with
``scale = max(amax / 448, 2^-100)``, so every value is within half an e4m3 step of the appended one
and no calibration is needed.  Half the bytes of a bf16 cache, plus 4 per row.  Since the scales
are indexed as the slots are, ``copy_accepted_kv`` commits both: the codes as any pool, the scales
as a pool of head size 1 (``scales.unsqueeze(-1)``).
"""
from __future__ import annotations

import ctypes

import torch

from . import _device, _lib
from .qk_norm import E4M3, check_scales


def store_kvcache_e4m3(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Quantise row i of key/value into cache slot ``slot_mapping[i]``; slot -1 skips the row.

    The e4m3 form of ``store_kvcache``: key and value are [rows, kv_heads, dim] in BF16, FP16 or
    FP32, any positive strides.  A row that holds an infinity or a NaN gets a NaN scale and zero
    codes (it reads as NaN).  Slots must be unique; one outside the cache writes nothing and records
    TV_STATUS_BAD_SLOT.
    """
    if key.ndim != 3 or value.shape != key.shape or key.dtype != value.dtype:
        raise ValueError("key and value must be [rows,heads,dim] of one shape and dtype")
    rows, heads, dim = key.shape
    if heads < 1 or not 2 <= dim <= 256 or dim % 2:
        raise ValueError("store_kvcache_e4m3 takes even head sizes from 2 to 256")
    if (k_cache.ndim != 4 or v_cache.shape != k_cache.shape or tuple(k_cache.shape[2:]) != (heads, dim)
            or k_cache.dtype != E4M3 or v_cache.dtype != E4M3 or k_cache.shape[0] < 1 or k_cache.shape[1] < 1):
        raise ValueError("caches must be float8_e4m3fn [pages,page_size,heads,dim]")
    check_scales(k_cache, k_scale, "k_scale")
    check_scales(v_cache, v_scale, "v_scale")
    if slot_mapping.ndim != 1 or slot_mapping.numel() != rows or slot_mapping.dtype not in (torch.int32, torch.int64):
        raise ValueError("slot_mapping must be an int32 or int64 [rows] vector")
    device = _device.require_gpu(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping, what="store_kvcache_e4m3")
    if rows == 0:
        return
    a = _lib.StoreE4m3Args()
    a.key, a.key_stride[:] = key.data_ptr(), key.stride()
    a.value, a.value_stride[:] = value.data_ptr(), value.stride()
    a.k_cache, a.k_cache_stride[:] = k_cache.data_ptr(), k_cache.stride()
    a.v_cache, a.v_cache_stride[:] = v_cache.data_ptr(), v_cache.stride()
    a.k_scale, a.k_scale_stride[:] = k_scale.data_ptr(), k_scale.stride()
    a.v_scale, a.v_scale_stride[:] = v_scale.data_ptr(), v_scale.stride()
    a.pool_pages, a.page_size = k_cache.shape[0], k_cache.shape[1]
    a.slots, a.slots_stride = slot_mapping.data_ptr(), slot_mapping.stride(0)
    a.slots_is_int64 = slot_mapping.dtype == torch.int64
    a.rows, a.kv_heads, a.head_dim, a.dtype = rows, heads, dim, _device.dtype_code(key.dtype)
    a.status = _device.status_word(device).data_ptr()
    code = _device.call(device, _lib.library().tv_store_kvcache_e4m3, ctypes.byref(a), _device.stream_handle(device))
    _lib.check(code, "store_kvcache_e4m3")
