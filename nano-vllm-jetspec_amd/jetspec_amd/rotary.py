"""The rotation of Q and K in the layouts ``rope_scatter`` does not have, with the K/V scatter.

The reference rotates the two halves of whole heads by angles from a table (tree_fusion.py:31-82,
layers/rotary_embedding.py:29-35).  Other models pair neighbouring dimensions, turn only the first part of
a head, or run beyond the lengths a table was made for with frequencies scaled down.  Here the angles come
from the positions and the frequencies, in 64 bits in the kernel (tv_rotary_scatter), so no table bounds
the positions and any scaling is a vector of frequencies (``rotary_frequencies``).
"""
from __future__ import annotations

import math

import torch

from . import _device, _lib
from .tree_fusion import _one_address_per_element, _share_bytes

_INDEX_DTYPES = (torch.int32, torch.int64)
_VALUE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, factor: float = 1.0, original_length: int | None = None,
                       slow: float = 1.0, fast: float = 32.0, ramp: str = "turns", device=None) -> torch.Tensor:
    """float64 [rotary_dim / 2] radians a position: ``base ** (-2p / rotary_dim)``, for ``factor`` times longer contexts.

    Without ``original_length`` all are divided by ``factor`` (positions interpolated).  With it, frequencies
    that turn more than ``fast`` times over that length stay, those below ``slow`` turns are divided, and those
    between are blended.  The blend is part of what a checkpoint was trained with, and the two in use differ by tens
    of percent: ``ramp="turns"`` is linear in a frequency's turns, ``ramp="pairs"`` in its index, between the
    index of ``fast`` turns rounded down and that of ``slow`` turns rounded up, as checkpoints with thresholds of 1 and 32
    mostly have it.  ``rotary_scatter`` takes a scaling's amplitude as ``gain``.
    """
    if isinstance(rotary_dim, bool) or not isinstance(rotary_dim, int) or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even int")
    if not 0 < base < math.inf or not 0 < factor < math.inf:
        raise ValueError("base and factor must be positive and finite")
    if ramp not in ("turns", "pairs"):
        raise ValueError("ramp must be 'turns' or 'pairs'")
    if ramp == "pairs" and (base <= 1 or slow <= 0):
        raise ValueError("a ramp over pairs needs a base above 1 and slow above 0")
    plain = torch.tensor([base ** (-2 * p / rotary_dim) for p in range(rotary_dim // 2)], dtype=torch.float64)
    if original_length is None:
        return (plain / factor).to(device)
    if original_length <= 0 or not 0 <= slow < fast < math.inf:
        raise ValueError("original_length must be positive, and slow below fast")
    if ramp == "turns":
        keep = ((plain * original_length / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
    else:
        # base ** (-2p / rotary_dim) turns t times over the length at this p.
        first, last = (rotary_dim * math.log(original_length / (2 * math.pi * t)) / (2 * math.log(base)) for t in (fast, slow))
        first, last = max(math.floor(first), 0), min(math.ceil(last), rotary_dim - 1)
        at = torch.arange(rotary_dim // 2, dtype=torch.float64)
        keep = ((last - at) / max(last - first, 1e-3)).clamp(0, 1)
    return (plain * (keep + (1 - keep) / factor)).to(device)


def _check_shapes(q, k, v, positions, frequencies, k_pool, v_pool, node_slots, out, gain) -> tuple[int, tuple, tuple]:
    """What the kernel's addresses rest on; no tensor value is read.  Returns the GPU's index and the
    shapes of q and the pools."""
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
    if (frequencies.ndim != 1 or frequencies.dtype is not torch.float64 or not 1 <= frequencies.shape[0] <= dim // 2
            or not frequencies.is_contiguous()):
        raise ValueError("frequencies must be a dense float64 vector of at most dim / 2")
    pool = k_pool.shape
    if (len(pool) != 4 or v_pool.shape != pool or pool[0] < 1 or pool[1] < 1 or pool[2] != kv_heads or pool[3] != dim
            or k_pool.dtype is not dtype or v_pool.dtype is not dtype):
        raise ValueError("KV pools must match [pages,page_size,kv_heads,dim] in the Q/K/V dtype")
    if not -3e38 <= gain <= 3e38:   # fp32 in the kernel
        raise ValueError("gain must be finite")
    if out is None:
        return _device.one_gpu("rotary_scatter", q, k, v, positions, frequencies, k_pool, v_pool, node_slots), shape, pool
    if out.shape != shape or out.dtype is not dtype:
        raise ValueError("output must match Q shape and dtype")
    return _device.one_gpu("rotary_scatter", q, k, v, positions, frequencies, k_pool, v_pool, node_slots, out), shape, pool


def _check_layouts(q, k, v, positions, frequencies, k_pool, v_pool, node_slots, out):
    """No two written elements share an address, and nothing written is read."""
    read, written = (q, k, v, positions, frequencies, node_slots), (k_pool, v_pool, out)
    if any(min(t.stride()) <= 0 for t in (*read, *written) if t.numel()):
        raise ValueError("rotary_scatter requires positive tensor strides")
    if not all(_one_address_per_element(t) for t in written):
        raise ValueError("written layouts must not have overlapping addresses")
    if any(_share_bytes(a, b) for i, a in enumerate(written) for b in written[i + 1:]):
        raise ValueError("output and pools must not overlap")
    if any(_share_bytes(a, b) for a in written for b in read if b.numel()):
        raise ValueError("output and pools must not overlap source tensors")


def rotary_scatter(q, k, v, positions, frequencies, k_pool, v_pool, node_slots, *, interleaved: bool = False,
                   gain: float = 1.0, out=None):
    """Validate, then return the rotated Q, scattering rotated K and raw V.

    With n frequencies, pair p of a head is ``(x[p], x[n + p])``, or ``(x[2p], x[2p + 1])`` if ``interleaved``; it is
    turned by ``positions * frequencies[p]`` and multiplied by ``gain``, and dimensions from 2n on are copied.
    Q, K and V are [rows, heads, dim] in BF16, FP16 or FP32, even dim up to 256, the pools [pages, page_size,
    kv_heads, dim] in their type; all may be strided.  FP32 throughout, rounded once when stored.  A node slot
    of -1 marks a padding row, which is left alone; the others must be in range and unique, positions in
    [0, 2^31).  This boundary checks the values of positions and slots on the device and therefore
    synchronises; a layer loop calls ``rotary_scatter_prevalidated``.
    """
    _check_shapes(q, k, v, positions, frequencies, k_pool, v_pool, node_slots, out, gain)
    if q.shape[0] < 1:
        raise ValueError("rotary_scatter needs at least one row")
    if out is None:
        out = torch.zeros_like(q)   # padding rows of a new output are zero
    _check_layouts(q, k, v, positions, frequencies, k_pool, v_pool, node_slots, out)
    kept = node_slots != -1
    live = node_slots[kept]
    if live.numel():
        low, high = torch.aminmax(positions[kept])
        if int(low) < 0 or int(high) > 0x7fffffff:
            raise ValueError("positions must lie in [0, 2^31)")
        low, high = torch.aminmax(live)
        if int(low) < 0 or int(high) >= k_pool.shape[0] * k_pool.shape[1]:
            raise ValueError("node slots lie outside the KV pool")
        if torch.unique(live).numel() < live.numel():
            raise ValueError("node slots must be unique to avoid KV write races")
    return rotary_scatter_prevalidated(q, k, v, positions, frequencies, k_pool, v_pool, node_slots, out,
                                       interleaved=interleaved, gain=gain)


def rotary_scatter_prevalidated(q, k, v, positions, frequencies, k_pool, v_pool, node_slots, out, *,
                                interleaved: bool = False, gain: float = 1.0):
    """Launch-only boundary: shapes and dtypes are checked, nothing is allocated or synchronised.

    The caller guarantees the layouts and values ``rotary_scatter`` checks.  The kernel still refuses to
    write for a position or slot out of range (status bits, read with ``read_and_clear_status``) instead of
    touching memory it does not own.
    """
    if out is None:
        raise ValueError("rotary_scatter_prevalidated writes to a given output")
    index, shape, pool = _check_shapes(q, k, v, positions, frequencies, k_pool, v_pool, node_slots, out, gain)
    if shape[0] == 0:
        return out
    args = _lib.pack_rotary(
        q.data_ptr(), *q.stride(), k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), positions.data_ptr(),
        positions.stride(0), positions.dtype is torch.int64, 0, 0, 0, 0, 0, k_pool.data_ptr(), *k_pool.stride(),
        v_pool.data_ptr(), *v_pool.stride(), pool[0], pool[1], node_slots.data_ptr(), node_slots.stride(0),
        node_slots.dtype is torch.int64, out.data_ptr(), *out.stride(), shape[0], shape[1], pool[2], shape[2],
        _device.dtype_code(q.dtype), _device.status_pointer(index), frequencies.data_ptr(), frequencies.shape[0],
        bool(interleaved), gain)
    code = _device.launch(index, _lib.library().tv_rotary_scatter, args)
    if code:
        _lib.check(code, "rotary_scatter")
    return out
