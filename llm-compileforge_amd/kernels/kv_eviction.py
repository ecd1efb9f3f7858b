"""Eviction from a paged KV cache by accumulated attention weight, on MI355X.

No counterpart in the reference, whose caches keep every token of a request
(python_runtime/engine/cache_manager.py:79-267).  A sequence's account is the
attention weight that each of its cached tokens has drawn, per KV head or once
for all heads: `paged_attention_weights` and `chunk_attention_weights`
(kernels/paged_attention.py) write it.  When a sequence outgrows its budget,

    keep, new_lens = evict_select(weights, seq_lens, budget, sink=4, recent=256, ...)
    evict_move(keep, seq_lens, block_tables, k_cache, v_cache, weights=weights, ...)

keeps its first tokens, its latest ones and the heaviest of the others, head
by head, in the first new_lens slots of its blocks; the blocks behind them are
free.  Attention does not depend on the order of the slots, so only tokens
past the new end move, into the slots of evicted ones.

After a sequence's first eviction its slots no longer follow its text.  Its
`positions` then say where each slot's token stands (they decide what is first
and what is latest), for the slots below `kept`; slots from there on hold the
tokens appended since, the last of them at position seen - 1.  A caller keeps
positions int32 [B, heads, slots], kept and seen int32 [B], sets kept to
new_lens after each eviction, and starts a new sequence in a row with kept 0.
"""

from __future__ import annotations

import torch

from cf_hip import ops as _ops


def evict_select(
    weights: torch.Tensor,
    seq_lens: torch.Tensor,
    budget: int,
    *,
    sink: int = 0,
    recent: int = 0,
    positions: torch.Tensor | None = None,
    kept: torch.Tensor | None = None,
    seen: torch.Tensor | None = None,
    keep: torch.Tensor | None = None,
    new_lens: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Which cached tokens each head keeps.

    Args:
        weights: float32 [B, H, S] accounts, one row a KV head, or H = 1.
        seq_lens: int32 [B] tokens in each cache.
        budget: tokens that stay (a sequence of no more keeps all).
        sink, recent: leading and latest positions that always stay;
            sink + recent <= budget.
        positions, kept, seen: int32 [B, H, S], [B], [B]; none of them as
            long as nothing was evicted (a slot's index is its position).
        keep, new_lens: outputs, allocated if not given; memory of their own
            (new_lens over seq_lens, kept or seen is refused: every head of a
            sequence reads them, and so does evict_move afterwards).

    Returns:
        (keep int32 [B, H, budget], new_lens int32 [B]): keep[b, h, j] is the
        slot whose token belongs in slot j, -1 for j >= new_lens[b].
    """
    return _ops.evict_select(weights, seq_lens, budget, sink, recent, positions, kept, seen, keep, new_lens)


def evict_move(
    keep: torch.Tensor,
    seq_lens: torch.Tensor,
    block_tables: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    weights: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    kept: torch.Tensor | None = None,
    seen: torch.Tensor | None = None,
) -> None:
    """Moves what `evict_select` kept into its slots, in place.

    Args:
        keep, seq_lens: evict_select's result and lengths.
        block_tables: int32 [B, Mb]; the blocks written must not be shared.
        k_cache, v_cache: [num_blocks, block_size, Hkv, D], any strides and
            dtype; FP8 codes move as they are.
        weights, positions, kept, seen: those given to evict_select; the
            slots' weights and positions move with their rows.
    """
    _ops.evict_move(keep, seq_lens, block_tables, k_cache, v_cache, weights, positions, kept, seen)


__all__ = ["evict_move", "evict_select"]
