"""Block tables and slot maps of a batch, built on the device from request lengths.

The reference keeps both on the host: pages are taken per request from a free list
(engine/block_manager.py:58-103), and every step loops over the requests to make the slot
mapping (engine/model_runner.py:172-188) or a packed batch's row maps
(packed_metadata.py:151-195) and uploads them.  Here each is one launch on torch's current
stream that reads the lengths on the device, so a serving loop whose lengths live there (or a
captured one) needs no host round trip:

  build_block_tables  lengths + held tables + free list -> the batch's page tables
  packed_slot_maps    cached and new lengths -> cu_seqlens, row maps, positions, slots
"""
from __future__ import annotations

import torch

from . import _device, _lib

_INDEX_DTYPES = (torch.int32, torch.int64)


def _narrow(tensor: torch.Tensor) -> torch.Tensor:
    """int32 values; what does not fit is the nearest that does, and too large or negative either way."""
    return tensor if tensor.dtype is torch.int32 else tensor.clamp(-1 << 31, (1 << 31) - 1).to(torch.int32)


def _narrow_places(tensor: torch.Tensor) -> torch.Tensor:
    """int32 cache lengths or depths: one too large for int32 becomes the lowest, since the nearest is a place
    that a row could have, and would map to without a word."""
    return tensor if tensor.dtype is torch.int32 else tensor.clamp(-1 << 31, 1 << 31).to(torch.int32)   # 2^31 wraps


def _vector(tensor: torch.Tensor, what: str, narrow=_narrow) -> torch.Tensor:
    """An integer vector as the kernels read it: dense int32."""
    if tensor.ndim != 1 or tensor.dtype not in _INDEX_DTYPES:
        raise ValueError(f"{what} must be an int32 or int64 vector")
    if tensor.dtype is torch.int32 and tensor.is_contiguous():
        return tensor
    return narrow(tensor).contiguous()


def _table(tensor: torch.Tensor, requests: int, what: str) -> torch.Tensor:
    if tensor.ndim != 2 or tensor.shape[0] != requests or tensor.dtype not in _INDEX_DTYPES:
        raise ValueError(f"{what} must be an int32 or int64 [requests, pages] table")
    if tensor.dtype is torch.int32 and tensor.is_contiguous():
        return tensor
    tensor = _narrow(tensor)
    return tensor if tensor.stride(1) == 1 and tensor.stride(0) >= tensor.shape[1] else tensor.contiguous()


def build_block_tables(lengths: torch.Tensor, free_pages: torch.Tensor, block_size: int, width: int, *,
                       held_tables: torch.Tensor | None = None, held_counts: torch.Tensor | None = None,
                       free_count: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The page tables of a batch whose requests are ``lengths`` tokens long.

    Request r needs ``ceil(lengths[r] / block_size)`` pages; it keeps the first ``held_counts[r]``
    entries of ``held_tables[r]`` (at most ``width`` columns) and takes the rest from
    ``free_pages``, in request order.  ``free_count`` (one integer on the device) is the free
    list's live length when the tensor is larger, as a captured batch's is.

    Returns ``(tables, counts, taken)``: int32 ``[requests, width]`` tables padded with -1, the
    pages each request holds now (never fewer than before), and the number of pages taken, always
    the first ones of the list.  A request whose pages would pass ``width`` gets none, and neither
    does any growing request from the first on that the list is short for: they keep what they held,
    ``counts[r] * block_size < lengths[r]`` tells which, and the status word records
    TV_STATUS_NO_PAGES.  Lengths below 0 and counts outside the table or list are clamped
    (TV_STATUS_BAD_REQUEST).  The inputs are only read.
    """
    block_size, width = int(block_size), int(width)
    if block_size < 1 or width < 1:
        raise ValueError("build_block_tables requires a positive block size and table width")
    if (held_tables is None) != (held_counts is None):
        raise ValueError("held_tables and held_counts come together")
    lengths, free_pages = _vector(lengths, "lengths"), _vector(free_pages, "free_pages")
    requests = int(lengths.numel())
    tensors = [lengths, free_pages]
    if held_tables is not None:
        held_tables, held_counts = _table(held_tables, requests, "held_tables"), _vector(held_counts, "held_counts")
        if held_counts.numel() != requests or held_tables.shape[1] > width:
            raise ValueError("held_tables and held_counts must match the requests and fit the table width")
        tensors += [held_tables, held_counts]
    if free_count is not None:
        free_count = _vector(free_count.reshape(-1), "free_count")
        if free_count.numel() != 1:
            raise ValueError("free_count is one integer")
        tensors.append(free_count)
    index = _device.one_gpu("build_block_tables", *tensors)
    device = lengths.device
    tables = torch.empty(requests, width, dtype=torch.int32, device=device)
    counts = torch.empty(requests, dtype=torch.int32, device=device)
    taken = torch.empty(1, dtype=torch.int32, device=device)
    held = (None, 0, 0, None) if held_tables is None else (held_tables.data_ptr(), held_tables.stride(0),
                                                           held_tables.shape[1], held_counts.data_ptr())
    code = _device.launch(
        index, _lib.library().tv_build_block_tables, lengths.data_ptr(), *held, free_pages.data_ptr(),
        None if free_count is None else free_count.data_ptr(), free_pages.numel(), requests, block_size, width,
        tables.data_ptr(), counts.data_ptr(), taken.data_ptr(), _device.status_pointer(index))
    if code:
        _lib.check(code, "build_block_tables")
    return tables, counts, taken


def packed_slot_maps(cache_lens: torch.Tensor, query_lens: torch.Tensor, total_rows: int, block_size: int,
                     num_blocks: int, *, block_tables: torch.Tensor | None = None,
                     arena_pages: torch.Tensor | None = None, depths: torch.Tensor | None = None
                     ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Row maps of a packed batch: ``query_lens[r]`` new rows behind ``cache_lens[r]`` cached tokens.

    Returns ``(cu_seqlens, query_to_request, query_local_row, positions, slots)``, int32 but for
    positions and slots (int64).  Row l of request r has position ``cache_lens[r] + l`` (with
    ``depths``, one per packed row: ``cache_lens[r] + depth``, as a draft tree's nodes have) and its
    K/V row lives either at that token's place in ``block_tables[r]`` (prefill chunks and decode
    tokens) or, with ``arena_pages``, at the packed row's place in the arena (draft trees in scratch
    pages).  ``total_rows`` sizes the outputs: rows behind the last request's are padding with
    request -1, position 0 and slot -1, which the appends skip.

    A page outside ``[0, num_blocks)`` or past the table or the arena gives slot -1 and records
    TV_STATUS_BAD_SLOT; negative cache lengths or positions, and int64 cache lengths or depths past
    int32, give slot -1 and record TV_STATUS_BAD_POSITION; negative query lengths (counted as 0) and
    batches of more than ``total_rows`` rows record TV_STATUS_BAD_REQUEST.
    """
    total_rows, block_size, num_blocks = int(total_rows), int(block_size), int(num_blocks)
    if total_rows < 0 or block_size < 1 or num_blocks < 1:
        raise ValueError("packed_slot_maps requires a row count, a positive block size and a positive pool size")
    if (block_tables is None) == (arena_pages is None):
        raise ValueError("packed_slot_maps maps through either block_tables or arena_pages")
    cache_lens, query_lens = _vector(cache_lens, "cache_lens", _narrow_places), _vector(query_lens, "query_lens")
    requests = int(cache_lens.numel())
    if query_lens.numel() != requests:
        raise ValueError("cache_lens and query_lens disagree on the request count")
    tensors = [cache_lens, query_lens]
    if block_tables is not None:
        block_tables = _table(block_tables, requests, "block_tables")
        tensors.append(block_tables)
    else:
        arena_pages = _vector(arena_pages, "arena_pages")
        tensors.append(arena_pages)
    if depths is not None:
        depths = _vector(depths, "depths", _narrow_places)
        if depths.numel() != total_rows:
            raise ValueError("depths needs one entry per packed row")
        tensors.append(depths)
    index = _device.one_gpu("packed_slot_maps", *tensors)
    device = cache_lens.device
    # One allocation for three vectors: each costs the host as much as a quarter of the launch.
    request, local, cu = torch.empty(2 * total_rows + requests + 1, dtype=torch.int32, device=device).split_with_sizes(
        (total_rows, total_rows, requests + 1))
    positions = torch.empty(total_rows, dtype=torch.int64, device=device)
    slots = torch.empty(total_rows, dtype=torch.int64, device=device)
    # An empty table or arena has no address, and every row of it is out of range.
    if block_tables is not None:
        pages = (block_tables.data_ptr() or cu.data_ptr(), block_tables.stride(0), block_tables.shape[1], None, 0)
    else:
        pages = (None, 0, 0, arena_pages.data_ptr() or cu.data_ptr(), arena_pages.numel())
    code = _device.launch(
        index, _lib.library().tv_packed_slot_maps, cache_lens.data_ptr(), query_lens.data_ptr(), *pages,
        None if depths is None else depths.data_ptr(), requests, total_rows, block_size, num_blocks, cu.data_ptr(),
        request.data_ptr(), local.data_ptr(), positions.data_ptr(), slots.data_ptr(), _device.status_pointer(index))
    if code:
        _lib.check(code, "packed_slot_maps")
    return cu, request, local, positions, slots
