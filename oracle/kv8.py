"""The 8-bit KV cache's numbers in float64 (CPU, testing only).

A row's scale is 2^e with the smallest e >= -110 for which max |x| <= 448 2^e;
its codes are x / 2^e rounded to the nearest e4m3 value, ties to even.
Non-finite elements: code 0 and a NaN scale."""
from __future__ import annotations

import numpy as np

MAX = 448.0
MIN_EXP = -110


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 value of |x| <= 448 (3 fraction bits down to 2^-6, then
    multiples of 2^-9); numpy's rint rounds ties to even."""
    _, e = np.frexp(np.maximum(np.abs(x), 2.0 ** -6))  # |x| = m 2^e, m in [1/2, 1)
    step = np.ldexp(1.0, e - 4)
    return np.rint(x / step) * step


def quantize_rows(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes as values, scales) of the rows x[..., D]."""
    x = np.asarray(x, dtype=np.float64)
    finite = np.isfinite(x)
    x0 = np.where(finite, x, 0.0)
    a = np.abs(x0).max(axis=-1)
    e = np.full(a.shape, MIN_EXP, dtype=np.int64)
    while True:
        low = a > MAX * np.ldexp(1.0, e)
        if not low.any():
            break
        e = e + low
    codes = round_e4m3(np.ldexp(x0, -e[..., None]))
    return codes, np.where(finite.all(axis=-1), np.ldexp(1.0, e), np.nan)


def values(codes: np.ndarray, scales: np.ndarray, which: int) -> np.ndarray:
    """codes [pages, H, D] and scales [H, pages, 2] as the cache's values
    (which: 0 K, 1 V)."""
    return codes * scales[:, :, which].T[:, :, None]
