"""Plain numpy models of the e4m3 cache rows (test oracles; no code of the package)."""
from __future__ import annotations

import numpy as np
import torch


def _values() -> np.ndarray:
    """The value of every code 0..255: sign, 4 exponent bits of bias 7, 3 fraction bits; 0x7F is NaN."""
    out = np.empty(256)
    for code in range(256):
        exponent, fraction = (code >> 3) & 15, code & 7
        size = fraction * 2.0 ** -9 if exponent == 0 else (8 + fraction) * 2.0 ** (exponent - 10)
        out[code] = -size if code & 128 else size
        if code & 127 == 127:
            out[code] = np.nan
    return out


VALUES = _values()


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest code of each value up to 448 in size, ties to the even code; the sign of a zero is kept."""
    size = np.abs(x.astype(np.float64))
    ladder = VALUES[:127]
    high = np.clip(np.searchsorted(ladder, size), 1, 126)
    low = high - 1
    middle = (ladder[low] + ladder[high]) / 2
    code = np.where(size > middle, high, np.where(size < middle, low, low + (low & 1)))
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def quantise(rows: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scales) of fp32 rows [..., dim] as the appends define them, in fp32 arithmetic."""
    rows = rows.astype(np.float32)
    finite = np.isfinite(rows).all(-1)
    kept = np.where(finite[..., None], rows, np.float32(0))
    scale = np.maximum(np.abs(kept).max(-1) / np.float32(448), np.float32(2.0 ** -100))
    codes = encode(kept * (np.float32(1) / scale)[..., None])
    codes = np.where(finite[..., None], codes, np.uint8(0))
    return codes, np.where(finite, scale, np.float32(np.nan))


def codes_of(pool: torch.Tensor) -> np.ndarray:
    return pool.contiguous().view(torch.uint8).cpu().numpy()


def dequantise(pool: torch.Tensor, scale: torch.Tensor) -> np.ndarray:
    """A pool's rows in 64 bits."""
    return VALUES[codes_of(pool)] * scale.double().cpu().numpy()[..., None]
