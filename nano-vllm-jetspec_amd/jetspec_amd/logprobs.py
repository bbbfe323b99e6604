"""What a serving answer says about its tokens: log probabilities, entropy and alternatives.

The reference answers with tokens alone (serving_ops.py:55-90 takes one argmax a row).  This reads the
target's logits once (tv_token_logprobs), of all rows or of the accepted ones, without a normalised copy
of them.
"""
from __future__ import annotations

import torch

from . import _device, _lib

_INDEX_DTYPES = (torch.int32, torch.int64)
_VALUE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MOST_TOP = 64


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, *, top: int = 0, rows: torch.Tensor | None = None):
    """``(logprobs, entropy, top_ids, top_logprobs)`` of rows of [logits_rows, vocab] BF16, FP16 or FP32 logits.

    Result row i is about logits row ``rows[i]`` (row i without ``rows``).  ``token_ids`` is [n] or [n, tokens]
    int32/int64 and ``logprobs`` float32 of its shape: the log probability of each, 0 for token -1 (none).
    ``entropy`` is float32 [n] in nats.  ``top_ids`` int64 and ``top_logprobs`` float32 [n, top] are the ``top``
    (at most 64) most likely tokens in descending order, ties to the lowest index, a NaN above all: its first
    column is ``greedy_argmax``.  Words at -inf have probability zero; a row with a NaN or +inf, or of only -inf, has
    NaN in its numbers.  A row index of -1 is padding: zeros, ids -1.  Other indices and tokens outside
    give NaN (ids -1) and record TV_STATUS_BAD_REQUEST.  Nothing synchronises.
    """
    if logits.ndim != 2 or logits.shape[1] < 1:
        raise ValueError("logits must be [rows, vocab]")
    held, vocab = logits.shape
    if logits.dtype not in _VALUE_DTYPES:
        raise ValueError("logits must be BF16, FP16 or FP32")
    shape = token_ids.shape
    if len(shape) not in (1, 2) or token_ids.dtype not in _INDEX_DTYPES:
        raise ValueError("token_ids must be an int32 or int64 [rows] or [rows, tokens] tensor")
    count = shape[0]
    if rows is None:
        if count != held:
            raise ValueError("token_ids must have one entry per logits row")
        index = _device.one_gpu("token_logprobs", logits, token_ids)
    else:
        if rows.shape != (count,) or rows.dtype not in _INDEX_DTYPES:
            raise ValueError("rows must be an int32 or int64 vector with one entry per result row")
        index = _device.one_gpu("token_logprobs", logits, token_ids, rows)
        if not rows.is_contiguous():
            rows = rows.contiguous()
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= min(MOST_TOP, vocab):
        raise ValueError("top must be an int from 0 to 64, at most the vocabulary")
    device = logits.device
    if logits.stride(1) != 1 or logits.stride(0) < vocab:
        logits = logits.contiguous()
    if not token_ids.is_contiguous():
        token_ids = token_ids.contiguous()
    logprobs = torch.empty(shape, dtype=torch.float32, device=device)
    entropy = torch.empty(count, dtype=torch.float32, device=device)
    top_ids = torch.empty(count, top, dtype=torch.int64, device=device)
    top_logprobs = torch.empty(count, top, dtype=torch.float32, device=device)
    if count == 0:
        return logprobs, entropy, top_ids, top_logprobs
    args = _lib.pack_token_logprobs(
        # One row may have any row stride and still be contiguous; none is then used.
        logits.data_ptr(), max(logits.stride(0), vocab), held, vocab, _device.dtype_code(logits.dtype),
        0 if rows is None else rows.data_ptr(), rows is not None and rows.dtype is torch.int64, token_ids.data_ptr(),
        token_ids.dtype is torch.int64, count, shape[1] if len(shape) == 2 else 1, top, logprobs.data_ptr(),
        entropy.data_ptr(), top_ids.data_ptr(), top_logprobs.data_ptr(), _device.compute_units(index),
        _device.status_pointer(index))
    lib = _lib.library()
    size = lib.tv_token_logprobs_workspace_bytes(args)
    if size < 0:
        _lib.check(size, "token_logprobs")
    # Scratch of this call (or of the graph being captured): no two launches share one.
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    code = _device.launch(index, lib.tv_token_logprobs, args, workspace.data_ptr() if size else None, size)
    if code:
        _lib.check(code, "token_logprobs")
    return logprobs, entropy, top_ids, top_logprobs
