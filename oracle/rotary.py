"""Rotary positions with several axes in float64 (no reference counterpart:
its models carry their own rotary arithmetic)."""

from __future__ import annotations

import numpy as np


def axis_of_pair(pairs: int, sections, order: str) -> list[int]:
    axes = len(sections)
    if order == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [j % axes if j < axes * sections[j % axes] else 0 for j in range(pairs)]


def rotate(x, positions, inv_freq, sections, order: str = "blocks", adjacent: bool = False, scale: float = 1.0):
    """(rotated rows, |x1| + |x2| of each element's pair) of x [T, H, D] under positions [axes, T]."""
    x = np.array(x, dtype=np.float64)
    out, size = x.copy(), np.zeros_like(x)
    pairs = len(inv_freq)
    for j, a in enumerate(axis_of_pair(pairs, sections, order)):
        i1, i2 = (2 * j, 2 * j + 1) if adjacent else (j, j + pairs)
        angle = np.asarray(positions[a], dtype=np.float64) * float(inv_freq[j])
        c, s = np.cos(angle)[:, None] * scale, np.sin(angle)[:, None] * scale
        out[..., i1] = x[..., i1] * c - x[..., i2] * s
        out[..., i2] = x[..., i2] * c + x[..., i1] * s
        size[..., i1] = size[..., i2] = (np.abs(x[..., i1]) + np.abs(x[..., i2])) * abs(scale)
    return out, size
