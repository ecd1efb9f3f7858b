"""Plain statement of eviction by accumulated attention weight (no reference
counterpart): which slots a head keeps, and where each kept token goes."""

from __future__ import annotations

import numpy as np


def slot_positions(n: int, positions, kept: int, seen: int) -> np.ndarray:
    """Positions of a sequence's n slots: stored below `kept`, then in order up to seen - 1."""
    if positions is None:
        return np.arange(n)
    at = seen - n + np.arange(n)
    at[: min(kept, n)] = positions[: min(kept, n)]
    return at


def select(weights, n: int, budget: int, sink: int = 0, recent: int = 0, positions=None, kept: int = 0, seen: int = 0):
    """(keep [budget], new length) of one head of one sequence of n tokens."""
    keep = np.full(budget, -1, dtype=np.int32)
    if n <= budget:
        keep[:n] = np.arange(n)
        return keep, n
    w = np.asarray(weights[:n], dtype=np.float64)
    pos = slot_positions(n, positions, kept, seen)
    end = n if positions is None else seen

    def order(i):  # protected first, then NaN, then by weight; equal ones by slot
        if pos[i] < sink or pos[i] >= end - recent:
            return (0, 0.0, i)
        return (1, 0.0, i) if np.isnan(w[i]) else (2, -w[i] + 0.0, i)

    chosen = set(sorted(range(n), key=order)[:budget])
    movers = [i for i in sorted(chosen) if i >= budget]
    for j in range(budget):
        keep[j] = j if j in chosen else movers.pop(0)
    assert not movers
    return keep, budget
