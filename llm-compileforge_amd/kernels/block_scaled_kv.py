"""Paged KV caches in 8 bits with a scale for each block of tokens and KV head.

No counterpart in the reference, whose FP8 caches have one scale a tensor
(compiler/quantize/fp8_kv_cache.py:66-93); this framework's other FP8 caches have
one for each layer and KV head, to be calibrated before the first write.  Here the
scales come with the rows: a block's scale is the least that its largest value
needs, head by head, so nothing is calibrated and no value is out of range.  Codes
are float8_e4m3fn (scales are powers of two) or int8, whose codes are the finer ones
within such a block: over N(0, 1) values 0.9 % of their root mean square, e4m3fn
2.6 %.

    k_cache, v_cache = alloc_kv_cache(num_blocks, 16, heads, dim, torch.int8, device)
    k_scale, v_scale = alloc_kv_scales(num_blocks, heads, device)
    write_kv_blocks(k_new, v_new, block_tables, seq_lens, k_cache, v_cache, k_scale, v_scale)
    out = paged_attention_tensors(q, k_cache, v_cache, block_tables, seq_lens, k_scale=k_scale, v_scale=v_scale)

`paged_attention`, `paged_attention_tensors` and `chunked_prefill_attention` read such
a cache where their k_scale and v_scale are [num_blocks, heads]; so does
cf_hip.ops.paged_gather.  A block is copied or moved together with its scales:
BlockManager.copy_blocks and move_blocks take them as two more tensors (and a paired
cache as the one tensor that cf_hip.layout.paired_storage gives).
"""

from __future__ import annotations

import torch

from cf_hip import ops as _ops
from cf_hip.layout import alloc_kv_scales


def write_kv_blocks(
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    *,
    q_start: torch.Tensor | None = None,
) -> None:
    """Writes new rows at the last positions of their sequences.

    Args:
        k_new, v_new: [T, Hkv, D] float32, float16 or bfloat16, any strides.
        block_tables: int32 [N, Mb]; the blocks written to must not be shared
            (BlockManager.prepare_writes).
        seq_lens: int32 [N], tokens of each sequence including its new rows.
        k_cache, v_cache: [num_blocks, block_size, Hkv, D] float8_e4m3fn or int8,
            any strides (cf_hip.layout.alloc_kv_cache).
        k_scale, v_scale: float32 [num_blocks, Hkv]; updated.
        q_start: int32 [N + 1], ascending: sequence n owns rows [q_start[n],
            q_start[n + 1]).  Without it every sequence has one row (N = T; none
            where its length is 0), as in a decode step.

    A row at offset 0 of a block starts the block anew, whatever it held.  A later
    row that its scale does not reach widens it, and the codes before it are
    rounded again: exactly for e4m3fn but for codes that become subnormal, by half
    a step of the new scale for int8.  A NaN or infinity makes the scale of its
    block and head NaN, with which the block's values read as NaN until it starts
    anew; so do those of a scale that a caller made negative or infinite.  Rows past
    the table, at negative positions or of blocks outside the cache are skipped.
    """
    if isinstance(block_tables, torch.Tensor) and block_tables.dtype != torch.int32:
        block_tables = block_tables.to(torch.int32)
    if isinstance(seq_lens, torch.Tensor) and seq_lens.dtype != torch.int32:
        seq_lens = seq_lens.to(torch.int32)
    if isinstance(q_start, torch.Tensor) and q_start.dtype != torch.int32:
        q_start = q_start.to(torch.int32)
    _ops.kv_write_blocks(k_new, v_new, block_tables, seq_lens, k_cache, v_cache, k_scale, v_scale, q_start)


__all__ = ["alloc_kv_scales", "write_kv_blocks"]
