"""Packed tree attention with a sliding window and first tokens that stay visible.

The reference's layers see their whole prefix (paged_backend.py:116-213).  Models with sliding-window
layers see the last ``window`` positions and, often, a few first ones (sinks) that keep the softmax
steady once the window has left them.  Their cache needs no other pages: those may have been given back,
and their table entries may hold anything.
"""
from __future__ import annotations

import torch

from . import _device, _lib
from .cache_e4m3 import _vector
from .tree_fusion import _one_address_per_element, _share_bytes

_MOST = 0x7fffffff


def packed_window_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, metadata, positions: torch.Tensor,
                            scale: float, num_queries_per_kv: int, *, window: int, sinks: int = 0,
                            output_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``packed_tree_attention`` in which the row at position P sees the keys at positions x with
    ``P - x < window`` or ``x < sinks``, of its request's prefix and of its ancestors.

    q is [rows, heads, dim] in BF16 or FP16, the pools [pages, page_size, kv_heads, dim] in its type, dim a
    multiple of 8 up to 256, ``metadata`` any ``PackedTreeMetadata`` (a tree of one node is a decode token,
    a chain tree a prefill chunk) and ``positions`` its rows' int32 or int64 positions: the request's prefix
    length plus the node's depth, as the rotation takes them.  One outside [prefix, prefix + node] is taken as
    the nearer end and records TV_STATUS_BAD_POSITION.  Finite ``qq_bias`` values are added to the scores.
    The result is new, or ``out``, in q's dtype or FP32; a row that sees no key is zero, one that no request
    counts (padding of a captured batch) is left as it was.  For a result in q's dtype each probability is rounded to
    it (BF16 2^-8, FP16 2^-11 of it) before it meets V; ``output_dtype=torch.float32`` keeps more (2^-26, 2^-23).
    A row that sees a NaN or infinity in V has NaN or keeps the infinity, in that dimension or in all.

    Every length, page and position is read on the device, so a captured call follows the staged metadata,
    and no state is kept between calls.  Requests that reach outside the batch, the bias or their table row
    record TV_STATUS_BAD_REQUEST (their rows are not written); pages and slots outside the pool record
    TV_STATUS_BAD_PAGE and are skipped.  Pages that no row sees are not looked up.
    """
    m, shape, pool, kind = metadata, q.shape, k_pool.shape, q.dtype
    if len(shape) != 3 or shape[0] != m.total_queries:
        raise ValueError("packed queries do not match the metadata")
    if len(pool) != 4 or v_pool.shape != pool or pool[1] != m.block_size:
        raise ValueError("packed K/V page geometry does not match metadata")
    rows, heads, dim = shape
    if kind is not torch.bfloat16 and kind is not torch.float16:
        raise ValueError("packed queries must be BF16 or FP16")
    if k_pool.dtype is not kind or v_pool.dtype is not kind:
        raise ValueError("packed queries and K/V pools must share dtype")
    q_strides = q.stride()
    if q_strides[2] != 1 or pool[3] != dim or not 8 <= dim <= 256 or dim % 8:
        raise ValueError("unsupported packed query/KV head geometry (head sizes are multiples of 8 up to 256)")
    if (isinstance(num_queries_per_kv, bool) or not isinstance(num_queries_per_kv, int) or num_queries_per_kv <= 0
            or heads != pool[2] * num_queries_per_kv):
        raise ValueError("invalid packed GQA head grouping")
    if isinstance(window, bool) or not isinstance(window, int) or not 1 <= window <= _MOST:
        raise ValueError("window must be an int of at least 1")
    if isinstance(sinks, bool) or not isinstance(sinks, int) or not 0 <= sinks <= _MOST:
        raise ValueError("sinks must be an int of at least 0")
    if not -2.3e38 <= scale <= 2.3e38:   # scale * log2(e) is fp32 in the kernel
        raise ValueError("scale must be finite, and its product with log2(e) in fp32")
    dtype = kind if output_dtype is None else output_dtype
    if dtype is not kind and dtype is not torch.float32:
        raise ValueError("output dtype must match the queries or be FP32")
    if positions.shape != (rows,) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be an int32 or int64 [rows] vector")
    if out is not None:
        if out.shape != shape or out.dtype is not dtype or out.stride(2) != 1:
            raise ValueError("out must be [rows,heads,dim] in the output dtype, its last dimension contiguous")
        if not _one_address_per_element(out) or any(_share_bytes(out, t) for t in (q, k_pool, v_pool, positions) if t.numel()):
            raise ValueError("out must not overlap itself, the queries, the pools or the positions")
        index = _device.one_gpu("packed_window_attention", q, k_pool, v_pool, positions, out)
    else:
        index = _device.one_gpu("packed_window_attention", q, k_pool, v_pool, positions)
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
    if out is None:
        out = torch.empty(rows, heads, dim, dtype=dtype, device=q.device)
    if rows == 0:
        return out
    if q_strides[0] % 8 or q_strides[1] % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)   # dense ones too: their start may be what is off
        q_strides = q.stride()
    if not positions.is_contiguous():
        positions = positions.contiguous()
    out_strides = out.stride()
    args = _lib.pack_window_attention(
        q.data_ptr(), q_strides[0], q_strides[1], _device.dtype_code(kind), k_pool.data_ptr(), v_pool.data_ptr(),
        *k_pool.stride(), *v_pool.stride(), pool[0], out.data_ptr(), out_strides[0], out_strides[1],
        _device.dtype_code(dtype), cu, prefixes, counts, tables.data_ptr(), tables.stride(0), width[1], slots, bias, offsets,
        m.qq_bias.numel(), positions.data_ptr(), positions.dtype is torch.int64, window, sinks, requests, rows, heads,
        pool[2], dim, pool[1], scale, _device.compute_units(index), _device.status_pointer(index))
    lib = _lib.library()
    size = lib.tv_window_attention_workspace_bytes(args)
    if size < 0:
        _lib.check(size, "packed_window_attention")
    # Scratch of this call (or of the graph being captured): no two launches share one.
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    code = _device.launch(index, lib.tv_window_attention, args, workspace.data_ptr() if size else None, size)
    if code:
        _lib.check(code, "packed_window_attention")
    return out
