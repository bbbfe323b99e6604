"""An 8-bit K/V cache: e4m3 rows with a scale per slot and head, and the operators on it.

``k_cache`` and ``v_cache`` are float8_e4m3fn [pages, page_size, kv_heads, dim]; ``k_scale`` and
``v_scale`` float32 [pages, page_size, kv_heads].  A row of one head reads as ``code * scale`` with
``scale = max(amax / 448, 2^-100)``, so every value is within half an e4m3 step of the appended one
and no calibration is needed.  Half the bytes of a bf16 cache, plus 4 per row.  Since the scales
are indexed as the slots are, ``copy_accepted_kv`` commits both: the codes as any pool, the scales
as a pool of head size 1 (``scales.unsqueeze(-1)``).  The appends fill pools of any even head size up to
256; the attention reads those of 64, 128 and 256.
"""
from __future__ import annotations

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
    shape, pool = key.shape, k_cache.shape
    if len(shape) != 3 or value.shape != shape or key.dtype is not value.dtype:
        raise ValueError("key and value must be [rows,heads,dim] of one shape and dtype")
    rows, heads, dim = shape
    if heads < 1 or not 2 <= dim <= 256 or dim % 2:
        raise ValueError("store_kvcache_e4m3 takes even head sizes from 2 to 256")
    if (len(pool) != 4 or v_cache.shape != pool or pool[2] != heads or pool[3] != dim or k_cache.dtype is not E4M3
            or v_cache.dtype is not E4M3 or pool[0] < 1 or pool[1] < 1):
        raise ValueError("caches must be float8_e4m3fn [pages,page_size,heads,dim]")
    k_strides, v_strides = check_scales(pool, k_scale, "k_scale"), check_scales(pool, v_scale, "v_scale")
    if slot_mapping.shape != (rows,) or slot_mapping.dtype not in (torch.int32, torch.int64):
        raise ValueError("slot_mapping must be an int32 or int64 [rows] vector")
    index = _device.one_gpu("store_kvcache_e4m3", key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
    if rows == 0:
        return
    args = _lib.pack_store_e4m3(
        key.data_ptr(), *key.stride(), value.data_ptr(), *value.stride(), k_cache.data_ptr(), *k_cache.stride(),
        v_cache.data_ptr(), *v_cache.stride(), k_scale.data_ptr(), *k_strides, v_scale.data_ptr(), *v_strides, pool[0],
        pool[1], slot_mapping.data_ptr(), slot_mapping.stride(0), slot_mapping.dtype is torch.int64, rows, heads, dim,
        _device.dtype_code(key.dtype), _device.status_pointer(index))
    code = _device.launch(index, _lib.library().tv_store_kvcache_e4m3, args)
    if code:
        _lib.check(code, "store_kvcache_e4m3")


def _vector(metadata, name: str, dtype: torch.dtype, size: int | None, index: int) -> int:
    """Address of a metadata buffer, which the kernel reads raw: type, density and size have to hold."""
    t = getattr(metadata, name)
    if t.dtype is not dtype or t.ndim != 1 or not t.is_contiguous() or (size is not None and t.numel() != size):
        raise ValueError(f"metadata.{name} must be a contiguous {dtype} vector of the batch's size")
    if t.get_device() != index:
        raise ValueError("packed attention requires CUDA queries, KV and metadata on one device")
    return t.data_ptr()


def packed_tree_attention_e4m3(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                               v_scale: torch.Tensor, metadata, scale: float, num_queries_per_kv: int, *,
                               output_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``packed_tree_attention`` over an e4m3 cache: one ragged launch with independent visibility.

    q is [rows, heads, dim] in BF16 or FP16, dim 64, 128 or 256; the pools are e4m3 with their scales
    and ``metadata`` is any ``PackedTreeMetadata`` (a tree of one node is a decode token, a chain tree
    a prefill chunk).  Any query group, page size and tree size; finite ``qq_bias`` values are added
    to the scores.  The result is new, in q's dtype or FP32; a row that sees no key is zero, one that no
    request counts (padding of a captured batch) is not written.  BF16
    results round each probability times its key's scale to BF16 once, FP16 ones keep it to 2^-17
    and FP32 ones to 2^-26: a BF16 result with less error is the FP32 one, rounded.

    Every length, page and slot is read on the device, so a captured call follows the staged
    metadata, and no state is kept between calls.  Requests that reach outside the batch, the bias
    or their table row record TV_STATUS_BAD_REQUEST (their rows are not written); pages and slots
    outside the pool record TV_STATUS_BAD_PAGE and are skipped.
    """
    m, shape, pool, kind = metadata, q.shape, k_pool.shape, q.dtype
    if len(shape) != 3 or shape[0] != m.total_queries:
        raise ValueError("packed queries do not match the metadata")
    if len(pool) != 4 or v_pool.shape != pool or pool[1] != m.block_size:
        raise ValueError("packed K/V page geometry does not match metadata")
    if k_pool.dtype is not E4M3 or v_pool.dtype is not E4M3:
        raise ValueError("packed_tree_attention_e4m3 takes float8_e4m3fn pools")
    k_strides, v_strides = check_scales(pool, k_scale, "k_scale"), check_scales(pool, v_scale, "v_scale")
    rows, heads, dim = shape
    q_strides = q.stride()
    if q_strides[2] != 1 or pool[3] != dim or dim not in (64, 128, 256):
        raise ValueError("unsupported packed query/KV head geometry (head sizes 64, 128 and 256)")
    if (isinstance(num_queries_per_kv, bool) or not isinstance(num_queries_per_kv, int) or num_queries_per_kv <= 0
            or heads != pool[2] * num_queries_per_kv):
        raise ValueError("invalid packed GQA head grouping")
    if kind is not torch.bfloat16 and kind is not torch.float16:
        raise ValueError("packed queries must be BF16 or FP16")
    if not -2.3e38 <= scale <= 2.3e38:   # scale * log2(e) is fp32 in the kernel
        raise ValueError("scale must be finite, and its product with log2(e) in fp32")
    dtype = kind if output_dtype is None else output_dtype
    if dtype is not kind and dtype is not torch.float32:
        raise ValueError("output dtype must match the queries or be FP32")
    index = _device.one_gpu("packed_tree_attention_e4m3", q, k_pool, v_pool, k_scale, v_scale)
    requests = m.num_requests
    cu = _vector(m, "cu_seqlens_q", torch.int32, requests + 1, index)
    prefixes = _vector(m, "prefix_lens", torch.int32, requests, index)
    counts = _vector(m, "node_counts", torch.int32, requests, index)
    slots = _vector(m, "tree_slots", torch.int64, rows, index)
    bias = _vector(m, "qq_bias", torch.float32, None, index)
    offsets = _vector(m, "qq_bias_offsets", torch.int64, requests + 1, index)
    tables = m.block_tables
    width = tables.shape
    if tables.dtype is not torch.int32 or len(width) != 2 or width[0] != requests or tables.stride(1) != 1:
        raise ValueError("metadata.block_tables must be int32 [requests, pages] with unit column stride")
    if tables.get_device() != index:
        raise ValueError("packed attention requires CUDA queries, KV and metadata on one device")
    out = torch.empty(rows, heads, dim, dtype=dtype, device=q.device)
    if rows == 0:
        return out
    if q_strides[0] % 8 or q_strides[1] % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)   # dense ones too: their start may be what is off
        q_strides = q.stride()
    args = _lib.pack_tree_attention_e4m3(
        q.data_ptr(), q_strides[0], q_strides[1], _device.dtype_code(kind), k_pool.data_ptr(), v_pool.data_ptr(),
        *k_pool.stride(), *v_pool.stride(), k_scale.data_ptr(), v_scale.data_ptr(), *k_strides, *v_strides, pool[0],
        out.data_ptr(), heads * dim, dim, _device.dtype_code(dtype), cu, prefixes, counts, tables.data_ptr(),
        tables.stride(0), width[1], slots, bias, offsets, m.qq_bias.numel(), requests, rows, heads, pool[2], dim, pool[1],
        scale, _device.compute_units(index), _device.status_pointer(index))
    lib = _lib.library()
    size = lib.tv_tree_attention_e4m3_workspace_bytes(args)
    if size < 0:
        _lib.check(size, "packed_tree_attention_e4m3")
    # Scratch of this call (or of the graph being captured): no two launches share one.
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    code = _device.launch(index, lib.tv_tree_attention_e4m3, args, workspace.data_ptr(), size)
    if code:
        _lib.check(code, "packed_tree_attention_e4m3")
    return out
