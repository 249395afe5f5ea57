"""4-bit quantise / dequantise on the CPU (oracle; test infrastructure only).

A (token, head) row of 256 bf16 values is held as 128 bytes of e2m1 codes (the
even dim in a byte's low half) and 8 e8m0 scales, one for every 32 dims. Written
from the formats' definitions, value by value: the scale is searched for, the
code is the nearest value of the list.
"""
from __future__ import annotations

import numpy as np

BLOCK = 32
ROW = 136
E_MIN, E_MAX = -120, 125


def e2m1_value(code: int) -> float:
    """Value of an e2m1 code: sign, two exponent bits (bias 1), one mantissa bit."""
    s = -1.0 if code & 8 else 1.0
    e, m = (code >> 1) & 3, code & 1
    return s * (m * 0.5 if e == 0 else (1 + m / 2) * 2.0 ** (e - 1))


POSITIVE = np.array([e2m1_value(c) for c in range(8)])


def scale_exponent(most: float) -> int:
    """The least e in [E_MIN, E_MAX] with most <= 7 * 2^e (E_MAX where there is none)."""
    for e in range(E_MIN, E_MAX):
        if most <= 7 * 2.0 ** e:
            return e
    return E_MAX


def nearest_code(y: np.ndarray) -> np.ndarray:
    """Codes of the nearest values, ties to the even code; -0 keeps its sign."""
    a = np.abs(y)
    d = np.abs(a[..., None] - POSITIVE)
    best = d.argmin(-1)
    nxt = np.minimum(best + 1, 7)
    tie = (np.take_along_axis(d, nxt[..., None], -1) ==
           np.take_along_axis(d, best[..., None], -1))[..., 0] & (nxt != best)
    code = np.where(tie & (best % 2 == 1), nxt, best)
    return (code | np.where(np.signbit(y), 8, 0)).astype(np.uint8)


def quantize_rows(x) -> np.ndarray:
    """Values [..., 256] (float64 of bf16) -> rows [..., 136] uint8."""
    x = np.asarray(x, dtype=np.float64)
    lead = x.shape[:-1]
    b = x.reshape(-1, BLOCK)
    codes = np.zeros(b.shape, dtype=np.uint8)
    scales = np.full(len(b), 255, dtype=np.uint8)
    fine = np.isfinite(b).all(-1)
    most, at = np.unique(np.abs(b[fine]).max(-1), return_inverse=True)
    e = np.array([scale_exponent(m) for m in most], dtype=np.int64)[at]
    codes[fine] = nearest_code(b[fine] * 2.0 ** -e[:, None].astype(np.float64))
    scales[fine] = e + 127
    codes = codes.reshape(*lead, 128, 2)
    return np.concatenate([codes[..., 0] | codes[..., 1] << 4,
                           scales.reshape(*lead, 8)], -1).astype(np.uint8)


_VALUES = np.array([e2m1_value(c) for c in range(16)])


def values(rows) -> np.ndarray:
    """Rows [..., 136] uint8 -> float64 values [..., 256]; NaN where the scale is 255."""
    rows = np.asarray(rows)
    codes = np.stack([rows[..., :128] & 15, rows[..., :128] >> 4], -1)
    x = _VALUES[codes].reshape(*rows.shape[:-1], 8, BLOCK)
    byte = rows[..., 128:].astype(np.float64)
    scale = np.where(byte == 255, np.nan, 2.0 ** (byte - 127))
    return (x * scale[..., None]).reshape(*rows.shape[:-1], 256)
