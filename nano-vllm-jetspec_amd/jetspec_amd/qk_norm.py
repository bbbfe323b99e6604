"""Per-head Q/K RMS norm, HF-order RoPE and the K/V scatter of a layer in one launch.

The reference normalises the queries and keys of a tree layer in two eager norms and then runs
its fused rotation and scatter (models/qwen3.py:193-265, tree_fusion.py:167-199).  Here the three
are one gfx950 kernel (tv_qk_norm_rope_scatter) that reads Q, K and V once and writes the rotated
Q to ``out`` and K and V to their slots, in the pools' own type or as e4m3 codes with a scale per
slot and head.  Everything between the read and the write is fp32, rounded once; the eager order
(and ``rope_scatter``) rounds after the norm and after every product.
"""
from __future__ import annotations

import torch

from . import _device, _lib
from .tree_fusion import _one_address_per_element, _share_bytes

_INDEX_DTYPES = (torch.int32, torch.int64)
_VALUE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
E4M3 = torch.float8_e4m3fn


def check_scales(shape, scale: torch.Tensor | None, what: str) -> tuple[int, ...]:
    """The fp32 scales [pages, page_size, kv_heads] beside an e4m3 pool of `shape`; returns their strides."""
    if scale is None or scale.dtype is not torch.float32 or scale.shape != shape[:3]:
        raise ValueError(f"{what} must be float32 [pages,page_size,kv_heads] beside its e4m3 pool")
    strides = scale.stride()
    if min(strides) <= 0:
        raise ValueError(f"{what} must have positive strides")
    return strides


def _check_shapes(q, k, v, q_weight, k_weight, positions, cache, k_pool, v_pool, node_slots, k_scale, v_scale, out,
                  eps) -> tuple[int, bool, tuple, tuple]:
    """What the kernel's addresses rest on; no tensor value is read.  Returns the GPU's index, whether the
    pools are e4m3, and the shapes of q and the pools."""
    shape, kv_shape, dtype = q.shape, k.shape, q.dtype
    if len(shape) != 3 or len(kv_shape) != 3 or v.shape != kv_shape:
        raise ValueError("Q/K/V must be [rows,heads,dim] with equal K/V geometry")
    rows, q_heads, dim = shape
    kv_rows, kv_heads, kv_dim = kv_shape
    if (q_heads < 1 or kv_rows != rows or kv_heads < 1 or kv_dim != dim or q_heads % kv_heads or not 2 <= dim <= 256
            or dim % 2):
        raise ValueError("invalid Q/K/V GQA or even head geometry")
    if dtype not in _VALUE_DTYPES or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("Q/K/V must share one of BF16, FP16 and FP32")
    if (positions.shape != (rows,) or node_slots.shape != (rows,) or positions.dtype not in _INDEX_DTYPES
            or node_slots.dtype not in _INDEX_DTYPES):
        raise ValueError("positions and node_slots must be integer [rows] vectors")
    turns = cache.shape
    if (len(turns) not in (2, 3) or (len(turns) == 3 and turns[1] != 1) or turns[-1] != dim or turns[0] < 1
            or cache.dtype not in (torch.bfloat16, torch.float32)):
        raise ValueError("cos/sin cache must be BF16/FP32 [positions,dim] or [positions,1,dim]")
    kind = q_weight.dtype
    if (q_weight.shape != (dim,) or k_weight.shape != (dim,) or k_weight.dtype is not kind
            or (kind is not dtype and kind is not torch.float32) or not q_weight.is_contiguous()
            or not k_weight.is_contiguous()):
        raise ValueError("norm weights must be dense [dim] vectors in FP32 or the Q/K/V dtype")
    pool, stored = k_pool.shape, k_pool.dtype
    e4m3 = stored is E4M3
    if (len(pool) != 4 or v_pool.shape != pool or pool[0] < 1 or pool[1] < 1 or pool[2] != kv_heads or pool[3] != dim
            or not (e4m3 or stored is dtype) or v_pool.dtype is not stored):
        raise ValueError("KV pools must match [pages,page_size,kv_heads,dim] in the Q/K/V dtype or float8_e4m3fn")
    if not e4m3 and (k_scale is not None or v_scale is not None):
        raise ValueError("scales belong to float8_e4m3fn pools")
    if out is not None and (out.shape != shape or out.dtype is not dtype):
        raise ValueError("output must match Q shape and dtype")
    if not 0.0 <= eps <= 3e38:   # fp32 in the kernel
        raise ValueError("eps must be finite and not negative")
    tensors = [q, k, v, q_weight, k_weight, positions, cache, k_pool, v_pool, node_slots]
    if e4m3:
        check_scales(pool, k_scale, "k_scale")
        check_scales(pool, v_scale, "v_scale")
        tensors += [k_scale, v_scale]
    if out is not None:
        tensors.append(out)
    return _device.one_gpu("qk_norm_rope_scatter", *tensors), e4m3, shape, pool


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
    if out is None:
        raise ValueError("qk_norm_rope_scatter_prevalidated writes to a given output")
    index, e4m3, shape, pool = _check_shapes(q, k, v, q_weight, k_weight, positions, cos_sin_cache, k_pool, v_pool,
                                             node_slots, k_scale, v_scale, out, eps)
    if shape[0] == 0:
        return out
    turn = cos_sin_cache.stride()
    scales = ((1, k_scale.data_ptr(), *k_scale.stride(), v_scale.data_ptr(), *v_scale.stride()) if e4m3
              else (0, 0, 0, 0, 0, 0, 0, 0, 0))
    args = _lib.pack_qk_norm(
        q.data_ptr(), *q.stride(), k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), positions.data_ptr(),
        positions.stride(0), positions.dtype is torch.int64, cos_sin_cache.data_ptr(), cos_sin_cache.shape[0], turn[0],
        turn[-1], _device.dtype_code(cos_sin_cache.dtype), k_pool.data_ptr(), *k_pool.stride(), v_pool.data_ptr(),
        *v_pool.stride(), pool[0], pool[1], node_slots.data_ptr(), node_slots.stride(0), node_slots.dtype is torch.int64,
        out.data_ptr(), *out.stride(), shape[0], shape[1], pool[2], shape[2], _device.dtype_code(q.dtype),
        _device.status_pointer(index), q_weight.data_ptr(), k_weight.data_ptr(), _device.dtype_code(q_weight.dtype), eps,
        *scales)
    code = _device.launch(index, _lib.library().tv_qk_norm_rope_scatter, args)
    if code:
        _lib.check(code, "qk_norm_rope_scatter")
    return out
