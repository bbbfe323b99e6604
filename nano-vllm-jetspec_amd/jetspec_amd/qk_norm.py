"""Per-head Q/K RMS norm, HF-order RoPE and the K/V scatter of a layer in one launch.

The reference normalises the queries and keys of a tree layer in two eager norms and then runs
its fused rotation and scatter (models/qwen3.py:193-265, tree_fusion.py:167-199).  Here the three
are one gfx950 kernel (tv_qk_norm_rope_scatter) that reads Q, K and V once and writes the rotated
Q to ``out`` and K and V to their slots, in the pools' own type or as e4m3 codes with a scale per
slot and head.  Everything between the read and the write is fp32, rounded once; the eager order
(and ``rope_scatter``) rounds after the norm and after every product.
"""
from __future__ import annotations

import ctypes

import torch

from . import _device, _lib
from .tree_fusion import _one_address_per_element, _share_bytes

_INDEX_DTYPES = (torch.int32, torch.int64)
_VALUE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
E4M3 = torch.float8_e4m3fn


def check_scales(pool: torch.Tensor, scale: torch.Tensor | None, what: str) -> None:
    """The fp32 scales [pages, page_size, kv_heads] beside an e4m3 pool."""
    if scale is None or scale.dtype != torch.float32 or scale.shape != pool.shape[:3]:
        raise ValueError(f"{what} must be float32 [pages,page_size,kv_heads] beside its e4m3 pool")
    if min(scale.stride()) <= 0:
        raise ValueError(f"{what} must have positive strides")


def _check_shapes(q, k, v, q_weight, k_weight, positions, cache, k_pool, v_pool, node_slots, k_scale, v_scale, out,
                  eps) -> torch.device:
    """What the kernel's addresses rest on; no tensor value is read.  Returns the device."""
    if q.ndim != 3 or k.ndim != 3 or v.shape != k.shape:
        raise ValueError("Q/K/V must be [rows,heads,dim] with equal K/V geometry")
    rows, q_heads, dim = q.shape
    if (q_heads < 1 or k.shape[0] != rows or k.shape[1] < 1 or k.shape[2] != dim or q_heads % k.shape[1]
            or not 2 <= dim <= 256 or dim % 2):
        raise ValueError("invalid Q/K/V GQA or even head geometry")
    if q.dtype not in _VALUE_DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("Q/K/V must share one of BF16, FP16 and FP32")
    if (tuple(positions.shape) != (rows,) or tuple(node_slots.shape) != (rows,)
            or positions.dtype not in _INDEX_DTYPES or node_slots.dtype not in _INDEX_DTYPES):
        raise ValueError("positions and node_slots must be integer [rows] vectors")
    if (cache.ndim not in (2, 3) or (cache.ndim == 3 and cache.shape[1] != 1) or cache.shape[-1] != dim
            or cache.shape[0] < 1 or cache.dtype not in (torch.bfloat16, torch.float32)):
        raise ValueError("cos/sin cache must be BF16/FP32 [positions,dim] or [positions,1,dim]")
    for weight in (q_weight, k_weight):
        if (tuple(weight.shape) != (dim,) or weight.dtype != q_weight.dtype or weight.dtype not in (q.dtype, torch.float32)
                or not weight.is_contiguous()):
            raise ValueError("norm weights must be dense [dim] vectors in FP32 or the Q/K/V dtype")
    if (k_pool.ndim != 4 or v_pool.shape != k_pool.shape or k_pool.shape[0] < 1 or k_pool.shape[1] < 1
            or tuple(k_pool.shape[2:]) != (k.shape[1], dim) or k_pool.dtype not in (q.dtype, E4M3)
            or v_pool.dtype != k_pool.dtype):
        raise ValueError("KV pools must match [pages,page_size,kv_heads,dim] in the Q/K/V dtype or float8_e4m3fn")
    tensors = [q, k, v, q_weight, k_weight, positions, cache, k_pool, v_pool, node_slots]
    if k_pool.dtype == E4M3:
        check_scales(k_pool, k_scale, "k_scale")
        check_scales(v_pool, v_scale, "v_scale")
        tensors += [k_scale, v_scale]
    elif k_scale is not None or v_scale is not None:
        raise ValueError("scales belong to float8_e4m3fn pools")
    if out is not None:
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("output must match Q shape and dtype")
        tensors.append(out)
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be finite and not negative")
    return _device.require_gpu(*tensors, what="qk_norm_rope_scatter")


def _check_layouts(q, k, v, q_weight, k_weight, positions, cache, k_pool, v_pool, node_slots, k_scale, v_scale, out):
    """No two written elements share an address, and nothing written is read."""
    read = (q, k, v, q_weight, k_weight, positions, cache, node_slots)
    written = [t for t in (k_pool, v_pool, k_scale, v_scale, out) if t is not None]
    if any(min(t.stride()) <= 0 for t in (*read, *written) if t.numel()):
        raise ValueError("qk_norm_rope_scatter requires positive tensor strides")
    if not all(_one_address_per_element(t) for t in written):
        raise ValueError("written layouts must not have overlapping addresses")
    if any(_share_bytes(a, b) for i, a in enumerate(written) for b in written[i + 1:]):
        raise ValueError("output, pools and scales must not overlap")
    if any(_share_bytes(a, b) for a in written for b in read if b.numel()):
        raise ValueError("output, pools and scales must not overlap source tensors")


def qk_norm_rope_scatter(q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool, node_slots, *,
                         eps: float = 1e-6, k_scale=None, v_scale=None, out=None):
    """Validate, then return the normed and rotated Q, scattering normed and rotated K and raw V.

    ``x * rsqrt(mean(x^2) + eps) * weight`` per head of Q and K (``q_weight``, ``k_weight``: [dim]),
    then the rotation by the cache row ``[cos_half | sin_half]`` of each row's position.  ``k_pool``
    and ``v_pool`` are [pages, page_size, kv_heads, dim] in Q's dtype, or float8_e4m3fn with
    ``k_scale``/``v_scale`` float32 [pages, page_size, kv_heads].  A node slot of -1 marks a padding
    row, which is left alone; the others must be in range and unique.  Q/K/V, addresses and pools
    may be strided.  This boundary checks the values of positions and slots on the device and
    therefore synchronises; a layer loop calls ``qk_norm_rope_scatter_prevalidated``.
    """
    _check_shapes(q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool, node_slots, k_scale, v_scale,
                  out, eps)
    if q.shape[0] < 1:
        raise ValueError("qk_norm_rope_scatter needs at least one row")
    if out is None:
        out = torch.zeros_like(q)   # padding rows of a new output are zero
    _check_layouts(q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool, node_slots, k_scale, v_scale,
                   out)
    kept = node_slots != -1
    live = node_slots[kept]
    if live.numel():
        low, high = torch.aminmax(positions[kept])
        if int(low) < 0 or int(high) >= cos_sin_cache.shape[0]:
            raise ValueError("RoPE positions lie outside the cos/sin cache")
        low, high = torch.aminmax(live)
        if int(low) < 0 or int(high) >= k_pool.shape[0] * k_pool.shape[1]:
            raise ValueError("node slots lie outside the KV pool")
        if torch.unique(live).numel() < live.numel():
            raise ValueError("node slots must be unique to avoid KV write races")
    return qk_norm_rope_scatter_prevalidated(q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool,
                                             node_slots, out, eps=eps, k_scale=k_scale, v_scale=v_scale)


def qk_norm_rope_scatter_prevalidated(q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool,
                                      node_slots, out, *, eps: float = 1e-6, k_scale=None, v_scale=None):
    """Launch-only boundary: shapes and dtypes are checked, nothing is allocated or synchronised.

    The caller guarantees the layouts and values ``qk_norm_rope_scatter`` checks.  The kernel still
    refuses to write for a position or slot out of range (status bits, read with
    ``read_and_clear_status``) instead of touching memory it does not own.
    """
    device = _check_shapes(q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool, node_slots, k_scale,
                           v_scale, out, eps)
    if q.shape[0] == 0:
        return out
    args = _lib.QkNormArgs()
    rope = args.rope
    rope.q, rope.k, rope.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    rope.q_stride[:], rope.k_stride[:], rope.v_stride[:] = q.stride(), k.stride(), v.stride()
    rope.positions, rope.positions_stride = positions.data_ptr(), positions.stride(0)
    rope.positions_is_int64 = positions.dtype == torch.int64
    rope.cache, rope.cache_rows = cos_sin_cache.data_ptr(), cos_sin_cache.shape[0]
    rope.cache_stride_row, rope.cache_stride_elem = cos_sin_cache.stride(0), cos_sin_cache.stride(-1)
    rope.cache_dtype = _device.dtype_code(cos_sin_cache.dtype)
    rope.k_pool, rope.v_pool = k_pool.data_ptr(), v_pool.data_ptr()
    rope.k_pool_stride[:], rope.v_pool_stride[:] = k_pool.stride(), v_pool.stride()
    rope.pool_pages, rope.page_size = k_pool.shape[0], k_pool.shape[1]
    rope.node_slots, rope.slots_stride = node_slots.data_ptr(), node_slots.stride(0)
    rope.slots_is_int64 = node_slots.dtype == torch.int64
    rope.out, rope.out_stride[:] = out.data_ptr(), out.stride()
    rope.rows, rope.q_heads, rope.kv_heads, rope.head_dim = q.shape[0], q.shape[1], k.shape[1], q.shape[2]
    rope.dtype = _device.dtype_code(q.dtype)
    rope.status = _device.status_word(device).data_ptr()
    args.q_weight, args.k_weight = q_weight.data_ptr(), k_weight.data_ptr()
    args.weight_dtype = _device.dtype_code(q_weight.dtype)
    args.eps = eps
    if k_pool.dtype == E4M3:
        args.pool_e4m3 = 1
        args.k_scale, args.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        args.k_scale_stride[:], args.v_scale_stride[:] = k_scale.stride(), v_scale.stride()
    code = _device.call(device, _lib.library().tv_qk_norm_rope_scatter, ctypes.byref(args),
                        _device.stream_handle(device))
    _lib.check(code, "qk_norm_rope_scatter")
    return out
