"""Rotary positions with one or several axes, on MI355X.

The reference has no rotary kernel: its traced models carry their own rotary
arithmetic ahead of the cache intercept (python_runtime/engine/
mlir_executor.py:369-419).  Here a step's new rows take one launch: the
queries rotated, the keys rotated and written with the values to their paged
slots, in the cache's layout and type (FP8 included).

Channel pair j of a row turns by the angle positions[a, t] * inv_freq[j], where
a is the pair's axis.  Text has one axis; images and video have three (time,
height, width), dealt to the pairs by `sections`:
  axis_order="blocks"  sections (16, 24, 24): pairs 0-15 axis 0, 16-39 axis 1,
                       40-63 axis 2;
  axis_order="cycled"  sections (24, 20, 20): pairs 1, 4, .. 58 axis 1, pairs 2,
                       5, .. 59 axis 2, the others axis 0.
A pair is channels (j, j + pairs), or (2j, 2j + 1) with interleaved=True;
channels past the last pair are left as they are (partial rotary).  Scaled
variants come in through inv_freq and rotary_scale, which multiplies the
rotated channels.  Angles are formed in 64 bits, so positions in the millions
lose nothing; results are rounded once, to the output's or the cache's type.
"""

from __future__ import annotations

import torch

from cf_hip import ops as _ops


def rotary(
    x: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    sections: tuple[int, ...] | None = None,
    axis_order: str = "blocks",
    interleaved: bool = False,
    rotary_scale: float = 1.0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Rotated rows.

    Args:
        x: [T, H, D] float32, float16 or bfloat16, any strides.
        positions: int32 or int64 [T], or [axes, T] (at most four axes).
        inv_freq: float32 [pairs], 2 * pairs <= D.
        sections: pairs of each axis, summing to len(inv_freq); may be left
            out with one axis.
        out: where to write ([T, H, D] in x's dtype; x itself is fine).
    """
    return _ops.rotary(x, positions, inv_freq, sections, axis_order, interleaved, rotary_scale, out)


def rotary_cache_write(
    q: torch.Tensor,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    sections: tuple[int, ...] | None = None,
    axis_order: str = "blocks",
    interleaved: bool = False,
    rotary_scale: float = 1.0,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Rotates a step's queries and keys and writes its keys and values.

    Args:
        q, k_new, v_new: [T, Hq, D], [T, Hkv, D], [T, Hkv, D] of one dtype.
        positions, inv_freq, sections, axis_order, interleaved, rotary_scale:
            as `rotary`.
        slot_mapping: int32 or int64 [T], block * block_size + offset of each
            row; slots outside the cache are skipped, slots must be distinct.
        k_cache, v_cache: [num_blocks, block_size, Hkv, D] in any layout of
            cf_hip.layout, float32, float16, bfloat16 or float8_e4m3fn.
        k_scale, v_scale: dequant scales [Hkv] or [1] of FP8 caches.
        out: where to write the queries (q itself is fine).

    Returns:
        The rotated queries [T, Hq, D].
    """
    return _ops.rotary_cache_write(q, k_new, v_new, positions, inv_freq, slot_mapping, k_cache, v_cache, sections,
                                   axis_order, interleaved, rotary_scale, k_scale, v_scale, out)


__all__ = ["rotary", "rotary_cache_write"]
