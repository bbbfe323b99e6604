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


_METADATA_VECTORS = (("cu_seqlens_q", torch.int32), ("prefix_lens", torch.int32), ("node_counts", torch.int32),
                     ("tree_slots", torch.int64), ("qq_bias", torch.float32), ("qq_bias_offsets", torch.int64))


def _check_metadata(metadata, device: torch.device) -> None:
    """The kernel reads these buffers raw: dtypes, density and sizes have to hold."""
    requests, rows = metadata.num_requests, metadata.total_queries
    sizes = (requests + 1, requests, requests, rows, None, requests + 1)
    for (name, dtype), size in zip(_METADATA_VECTORS, sizes):
        t = getattr(metadata, name)
        if t.dtype != dtype or t.ndim != 1 or not t.is_contiguous() or (size is not None and t.numel() != size):
            raise ValueError(f"metadata.{name} must be a contiguous {dtype} vector of the batch's size")
        if t.device != device:
            raise ValueError("packed attention requires CUDA queries, KV and metadata on one device")
    tables = metadata.block_tables
    if tables.dtype != torch.int32 or tables.ndim != 2 or tables.shape[0] != requests or tables.stride(1) != 1:
        raise ValueError("metadata.block_tables must be int32 [requests, pages] with unit column stride")
    if tables.device != device:
        raise ValueError("packed attention requires CUDA queries, KV and metadata on one device")


def packed_tree_attention_e4m3(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                               v_scale: torch.Tensor, metadata, scale: float, num_queries_per_kv: int, *,
                               output_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``packed_tree_attention`` over an e4m3 cache: one ragged launch with independent visibility.

    q is [rows, heads, dim] in BF16 or FP16, dim 64, 128 or 256; the pools are e4m3 with their scales
    and ``metadata`` is any ``PackedTreeMetadata`` (a tree of one node is a decode token, a chain tree
    a prefill chunk).  Any query group, page size and tree size; finite ``qq_bias`` values are added
    to the scores.  The result is new, in q's dtype or FP32; a row that sees no key is zero.  BF16
    results round each probability times its key's scale to BF16 once, FP16 ones keep it to 2^-17
    and FP32 ones to 2^-26.

    Every length, page and slot is read on the device, so a captured call follows the staged
    metadata, and no state is kept between calls.  Requests that reach outside the batch, the bias
    or their table row record TV_STATUS_BAD_REQUEST (their rows are not written); pages and slots
    outside the pool record TV_STATUS_BAD_PAGE and are skipped.
    """
    if q.ndim != 3 or q.shape[0] != metadata.total_queries:
        raise ValueError("packed queries do not match the metadata")
    if k_pool.ndim != 4 or k_pool.shape != v_pool.shape or k_pool.shape[1] != metadata.block_size:
        raise ValueError("packed K/V page geometry does not match metadata")
    if k_pool.dtype != E4M3 or v_pool.dtype != E4M3:
        raise ValueError("packed_tree_attention_e4m3 takes float8_e4m3fn pools")
    check_scales(k_pool, k_scale, "k_scale")
    check_scales(v_pool, v_scale, "v_scale")
    rows, heads, dim = q.shape
    kv_heads = k_pool.shape[2]
    if q.stride(-1) != 1 or k_pool.shape[3] != dim or dim not in (64, 128, 256):
        raise ValueError("unsupported packed query/KV head geometry (head sizes 64, 128 and 256)")
    if (isinstance(num_queries_per_kv, bool) or not isinstance(num_queries_per_kv, int) or num_queries_per_kv <= 0
            or heads != kv_heads * num_queries_per_kv):
        raise ValueError("invalid packed GQA head grouping")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("packed queries must be BF16 or FP16")
    dtype = q.dtype if output_dtype is None else output_dtype
    if dtype not in (q.dtype, torch.float32):
        raise ValueError("output dtype must match the queries or be FP32")
    device = _device.require_gpu(q, k_pool, v_pool, k_scale, v_scale, what="packed_tree_attention_e4m3")
    _check_metadata(metadata, device)
    out = torch.empty((rows, heads, dim), dtype=dtype, device=device)
    if rows == 0:
        return out
    if q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.contiguous()
    m, tables = metadata, metadata.block_tables
    args = _lib.TreeAttentionE4m3Args(
        q.data_ptr(), q.stride(0), q.stride(1), _device.dtype_code(q.dtype), k_pool.data_ptr(), v_pool.data_ptr(),
        k_pool.stride(), v_pool.stride(), k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(), v_scale.stride(),
        k_pool.shape[0], out.data_ptr(), out.stride(0), out.stride(1), _device.dtype_code(dtype),
        m.cu_seqlens_q.data_ptr(), m.prefix_lens.data_ptr(), m.node_counts.data_ptr(), tables.data_ptr(),
        tables.stride(0), tables.shape[1], m.tree_slots.data_ptr(), m.qq_bias.data_ptr(), m.qq_bias_offsets.data_ptr(),
        m.qq_bias.numel(), m.num_requests, rows, heads, kv_heads, dim, m.block_size, scale,
        _device.compute_units(device.index), _device.status_word(device).data_ptr())
    lib = _lib.library()
    size = lib.tv_tree_attention_e4m3_workspace_bytes(args)
    _lib.check(min(size, 0), "packed_tree_attention_e4m3")
    # Scratch of this call (or of the graph being captured): no two launches share one.
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    code = _device.call(device, lib.tv_tree_attention_e4m3, args, workspace.data_ptr(), size,
                        _device.stream_handle(device))
    _lib.check(code, "packed_tree_attention_e4m3")
    return out
