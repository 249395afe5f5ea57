"""The norm of query and key heads and the rotation by position, in float64
(oracle; test infrastructure only): the formulas of
muserve/model/qwen35_layer_v2.py:458-469, dim by dim."""
from __future__ import annotations

import numpy as np


def norm_rope(x, positions, inv_freq, weight=None, eps=1e-6, rope_scale=1.0, zero_centered=False,
              interleaved=False):
    """x [T, H, D] -> (out [T, H, D], size [T, H, D]): size is what an output is
    made of, |y_i c| + |y_j s| (its rounding errors scale with it)."""
    x = np.asarray(x, dtype=np.float64)
    y = x
    if weight is not None:
        w = np.asarray(weight, dtype=np.float64) + (1.0 if zero_centered else 0.0)
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    inv_freq = np.asarray(inv_freq, dtype=np.float64)
    half = len(inv_freq)
    out, size = y.copy(), np.abs(y)
    for i in range(half):
        angle = np.asarray(positions, dtype=np.float64) * inv_freq[i]
        c = (rope_scale * np.cos(angle))[:, None]
        s = (rope_scale * np.sin(angle))[:, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        size[..., a] = np.abs(y[..., a] * c) + np.abs(y[..., b] * s)
        size[..., b] = np.abs(y[..., b] * c) + np.abs(y[..., a] * s)
    return out, size
