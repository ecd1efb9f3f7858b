"""Eviction without a GPU: what its entry points refuse, and the plain
statement itself."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cf_hip import _abi
from kernels.kv_eviction import evict_move, evict_select
from oracle import kv_eviction as oracle


def test_cpu_tensors_are_refused():
    w, n = torch.zeros(1, 2, 32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm"):
        evict_select(w, n, 8)
    k = torch.zeros(4, 16, 2, 64)
    with pytest.raises(ValueError, match="ROCm"):
        evict_move(torch.zeros(1, 2, 8, dtype=torch.int32), n, torch.zeros(1, 2, dtype=torch.int32), k, k)


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _select(**change):
    a = dict(weights=torch.zeros(2, 4, 64), seq_lens=_i32(2), positions=_i32(2, 4, 64), kept=_i32(2), seen=_i32(2),
             keep=_i32(2, 4, 16), new_lens=_i32(2), sink=1, recent=2)
    a.update(change)
    d = {n: None if a[n] is None else _abi.descriptor(a[n])
         for n in ("weights", "seq_lens", "positions", "kept", "seen", "keep", "new_lens")}
    for x in d.values():
        if x is not None:
            x.t.device = _abi.SFA_ROCM  # reach the checks; every call here is refused before a launch
    r = {n: _abi.ref(x) for n, x in d.items()}
    return _abi.lib().cf_evict_select(r["weights"], r["seq_lens"], r["positions"], r["kept"], r["seen"], a["sink"],
                                      a["recent"], r["keep"], r["new_lens"], None)


@pytest.mark.parametrize("change, message", [
    (dict(weights=torch.zeros(2, 4, 64, dtype=torch.float16)), "weights: expected f32"),
    (dict(weights=torch.zeros(2, 4)), "weights: expected rank 3"),
    (dict(weights=torch.zeros(2, 4, 128)[:, :, ::2]), "the last stride must be 1"),
    (dict(weights=torch.zeros(2, 1, 64).expand(2, 4, 64)), "rows overlap"),
    (dict(weights=torch.as_strided(torch.zeros(1024), (2, 4, 64), (96, 64, 1))), "rows overlap"),
    (dict(weights=torch.as_strided(torch.zeros(1024), (2, 4, 64), (64, 96, 1))), "rows overlap"),
    (dict(seq_lens=_i32(3)), "seq_lens has 3 entries"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "seq_lens: expected i32"),
    (dict(positions=None), "go together"),
    (dict(seen=None), "go together"),
    (dict(positions=_i32(2, 4, 63)), "positions has 63 slots"),
    (dict(positions=_i32(2, 3, 64)), "positions: size 3"),
    (dict(kept=_i32(1)), "kept has 1 entries"),
    (dict(keep=_i32(2, 3, 16)), "keep must be"),
    (dict(keep=_i32(2, 4, 0)), "budget must be positive"),
    (dict(keep=_i32(2, 1, 16).expand(2, 4, 16)), "keep: rows overlap"),
    (dict(new_lens=_i32(1)), "new_lens"),
    (dict(sink=-1), "sink"),
    (dict(sink=10, recent=7), "fit the budget"),
    (dict(sink=2**31 - 1, recent=2**31 - 1), "fit the budget"),
])
def test_select_refuses(change, message):
    assert _select(**change) == _abi.CF_ERR_INVALID
    assert message in _abi.last_error()


LENS, STATE = _i32(2), _i32(2, 3)


@pytest.mark.parametrize("change", [
    dict(seq_lens=LENS, new_lens=LENS),
    dict(kept=LENS, new_lens=LENS),
    dict(seen=LENS, new_lens=LENS),
    dict(seen=STATE[:, 1], new_lens=STATE[:, 1]),
    dict(kept=STATE.view(-1)[:2], new_lens=STATE.view(-1)[1:3]),  # one entry in common
    dict(seq_lens=STATE.view(-1)[::3], new_lens=STATE.view(-1)[3:5]),
    dict(seq_lens=LENS[:1].expand(2), new_lens=LENS),
    dict(seq_lens=LENS, new_lens=LENS, positions=None, kept=None, seen=None),
])
def test_select_refuses_new_lengths_over_what_its_heads_read(change):
    """One head's workgroup would write a length before another's has read the old one."""
    assert _select(**change) == _abi.CF_ERR_INVALID
    assert "new_lens must not share" in _abi.last_error()


def test_select_refuses_new_lengths_that_are_one():
    assert _select(new_lens=_i32(1).expand(2)) == _abi.CF_ERR_INVALID
    assert "new_lens: rows overlap" in _abi.last_error()


def test_select_takes_columns_of_one_tensor():
    """Lengths side by side in one tensor share no entry (no heads: nothing is launched)."""
    no_heads = dict(weights=torch.zeros(2, 0, 64), positions=_i32(2, 0, 64), keep=_i32(2, 0, 16))
    assert _select(seq_lens=STATE[:, 0], kept=STATE[:, 1], new_lens=STATE[:, 2], **no_heads) == 0, _abi.last_error()
    assert _select(seen=STATE.view(-1)[::3], new_lens=STATE.view(-1)[1:3], **no_heads) == 0, _abi.last_error()


def _move(**change):
    a = dict(keep=_i32(2, 4, 16), seq_lens=_i32(2), tables=_i32(2, 3), k=torch.zeros(9, 16, 4, 64),
             v=torch.zeros(9, 16, 4, 64), weights=torch.zeros(2, 4, 48), positions=_i32(2, 4, 48), kept=_i32(2),
             seen=_i32(2))
    a.update(change)
    d = [None if t is None else _abi.descriptor(t) for t in a.values()]
    for x in d:
        if x is not None:
            x.t.device = _abi.SFA_ROCM
    return _abi.lib().cf_evict_move(*(_abi.ref(x) for x in d), None)


@pytest.mark.parametrize("change, message", [
    (dict(keep=_i32(2, 3, 16)), "one account a KV head, or one for all"),
    (dict(keep=torch.zeros(2, 4, 16)), "keep: expected i32"),
    (dict(tables=_i32(3, 3)), "block_tables has 3 rows"),
    (dict(tables=torch.zeros(2, 3, dtype=torch.int64)), "block_tables: expected i32"),
    (dict(k=torch.zeros(9, 16, 4, 64, dtype=torch.int32)), "k_cache: dtype"),
    (dict(v=torch.zeros(9, 16, 4, 64, dtype=torch.float16)), "v_cache dtype"),
    (dict(v=torch.zeros(9, 16, 4, 32)), "v_cache shape"),
    (dict(weights=torch.zeros(2, 1, 48)), "weights must be"),
    (dict(positions=None), "go together"),
    (dict(positions=_i32(1, 4, 48)), "positions: size 1"),
    (dict(seq_lens=_i32(1)), "seq_lens has 1"),
])
def test_move_refuses(change, message):
    assert _move(**change) == _abi.CF_ERR_INVALID
    assert message in _abi.last_error()


def test_moves_into_two_thousand_million_slots_are_refused():
    d = torch.zeros(9, 16, 4, 64)
    big = _abi.descriptor(d)
    a = [_abi.descriptor(t) for t in (_i32(2, 4, 16), _i32(2), _i32(2, 3))]
    for x in (big, *a):
        x.t.device = _abi.SFA_ROCM
    big.t.r4.sizes[0] = 1 << 28
    assert _abi.lib().cf_evict_move(*(_abi.ref(x) for x in a), _abi.ref(big), _abi.ref(big), None, None, None, None,
                                    None) == _abi.CF_ERR_INVALID
    assert "too many cache slots" in _abi.last_error()


def test_the_plain_statement():
    w = np.array([5.0, 1.0, 9.0, 1.0, 7.0, 0.0, 9.0, 2.0])
    keep, n = oracle.select(w, 8, 4)
    assert n == 4 and keep.tolist() == [0, 4, 2, 6]
    assert oracle.select(w, 8, 4, sink=2, recent=1)[0].tolist() == [0, 1, 2, 7]
    assert oracle.select(w, 3, 4)[0].tolist() == [0, 1, 2, -1]
    assert oracle.select(np.ones(6), 6, 3)[0].tolist() == [0, 1, 2]
    assert oracle.select(np.array([1.0, np.nan, np.inf]), 3, 1)[0].tolist() == [1]
    # slot 0 holds the newest position: kept as recent
    assert oracle.select(np.zeros(4), 4, 2, recent=1, positions=np.array([9, 3, 4]), kept=3, seen=11)[0].tolist() == [0, 3]


# ── the block pool behind an eviction ──────────────────────


def test_truncate_gives_the_last_blocks_back():
    from python_runtime.engine.block_manager import BlockManager

    bm = BlockManager(16, 4)
    bm.bind_rows(4, 8)
    a = bm.allocate("a", 22)  # six blocks, the last half full
    bm.set_len("a", 22)
    bm.share_prefix("a", "b", 12)
    bm.set_len("b", 12)
    table, lens = np.full((4, 8), -1, np.int32), np.zeros(4, np.int32)

    def sync():
        for r, c, v, _ in bm.table_deltas():
            if c < 0:
                lens[r] = v
            else:
                table[r, c] = v

    sync()
    bm.truncate("a", 9)  # shared blocks 0-2 stay, 3-5 are free
    assert bm.get_blocks("a") == a[:3] and bm.num_free_blocks() == 13
    sync()
    row = bm.row_of("a")
    assert lens[row] == 9 and table[row].tolist() == a[:3] + [-1] * 5
    bm.truncate("a", 4)  # b still holds blocks 1 and 2
    assert bm.num_free_blocks() == 13 and bm.ref_count(a[1]) == 1 and bm.get_blocks("b") == a[:3]
    bm.truncate("a", 4)
    bm.truncate("b", 0)
    assert bm.get_blocks("b") == [] and bm.num_free_blocks() == 15 and bm.ref_count(a[0]) == 1
    sync()
    assert lens[bm.row_of("b")] == 0 and (table[bm.row_of("b")] == -1).all()
    slots, copies = bm.prepare_writes([("a", 4, 5)])  # a grows again from its new end
    assert len(copies) == 0 and len(bm.get_blocks("a")) == 3 and len(slots) == 5
    sync()
    assert lens[row] == 9 and table[row, :3].tolist() == bm.get_blocks("a")
    bm.free("a")
    bm.free("b")
    assert bm.num_free_blocks() == 16


def test_only_requests_over_the_budget_give_up_what_they_share():
    """The order of an eviction on the pool: copy-on-write for the requests that are cut, no others, and
    the next token in the slot behind the budget."""
    from python_runtime.engine.block_manager import BlockManager

    bm, budget = BlockManager(32, 4), 8
    bm.allocate("a", 0)
    bm.prepare_writes([("a", 0, 8)])
    for r in ("b", "c"):
        bm.share_prefix("a", r, 8)
        bm.set_len(r, 8)
    length = {"a": 8, "b": 8, "c": 8}
    bm.prepare_writes([("c", 8, 6)])
    length["c"] = 14
    free = bm.num_free_blocks()
    over = [r for r, n in length.items() if n > budget]
    assert over == ["c"]
    _, copies = bm.prepare_writes([(r, 0, budget) for r in over])
    assert len(copies) == 2 and bm.num_free_blocks() == free - 2  # c's two shared blocks
    assert bm.get_blocks("a") == bm.get_blocks("b")               # these two still share theirs
    assert not set(bm.get_blocks("c")) & set(bm.get_blocks("a"))
    for r in over:
        bm.truncate(r, budget)
        length[r] = budget
    assert bm.num_free_blocks() == free  # two blocks taken, two given back
    slots, copies = bm.prepare_writes([(r, length[r], 1) for r in over])
    assert len(copies) == 0 and slots.tolist() == [bm.get_blocks("c")[2] * 4]
    # at the length from before the cut it would be a gap of five slots
    assert len(bm.get_blocks("c")) == 3


def test_truncate_refuses():
    from python_runtime.engine.block_manager import BlockManager

    bm = BlockManager(8, 4)
    bm.allocate("a", 10)
    with pytest.raises(KeyError):
        bm.truncate("nobody", 1)
    with pytest.raises(ValueError, match="not 13 tokens"):
        bm.truncate("a", 13)
    with pytest.raises(ValueError, match="non-negative"):
        bm.truncate("a", -1)
    assert len(bm.get_blocks("a")) == 3
    bm.truncate("a", 12)
    assert len(bm.get_blocks("a")) == 3


def test_truncate_over_many_steps_keeps_the_pool_whole():
    import random

    from python_runtime.engine.block_manager import BlockManager

    bm, rng, bs = BlockManager(64, 4), random.Random(2), 4
    held: dict[str, int] = {}
    for step in range(400):
        rid = f"r{rng.randrange(6)}"
        if rid not in held:
            src = rng.choice(list(held)) if held and rng.random() < 0.5 else None
            if src:
                held[rid] = rng.randint(0, held[src])
                bm.share_prefix(src, rid, held[rid])
            else:
                held[rid] = 0
                bm.allocate(rid, 0)
            bm.set_len(rid, held[rid])
        elif rng.random() < 0.3:
            held[rid] = rng.randint(0, held[rid])
            bm.truncate(rid, held[rid])
        elif rng.random() < 0.1:
            bm.free(rid)
            del held[rid]
        elif held[rid] < 24:
            n = rng.randint(1, 6)
            bm.prepare_writes([(rid, held[rid], n)])
            held[rid] += n
        tables = [bm.get_blocks(r) for r in held]
        assert [len(t) for t in tables] == [-(-n // bs) for n in held.values()]
        used = {}
        for t in tables:
            assert len(set(t)) == len(t)
            for blk in t:
                used[blk] = used.get(blk, 0) + 1
        assert bm.num_free_blocks() == 64 - len(used)
        assert all(bm.ref_count(blk) == used.get(blk, 0) for blk in range(64))


def test_backend_ops_check_their_inputs():
    from python_runtime.hal.hip_backend import HipBackend

    be, x = HipBackend(), torch.zeros(2, 2, 64)
    names = {"rotary": 3, "rotary_cache_write": 8, "paged_attention_weights": 6, "chunk_attention_weights": 6,
             "cache_evict": 5}
    assert set(names) <= set(HipBackend.supported_ops())
    for name, n in names.items():
        with pytest.raises(ValueError, match=f"at least {n}"):
            be.execute(name, [x] * (n - 1))
        with pytest.raises(ValueError, match="at most"):
            be.execute(name, [x] * 9)
        with pytest.raises(ValueError, match="ROCm"):
            be.execute(name, [x] * n, budget=4)
    with pytest.raises(ValueError, match="budget"):
        be.execute("cache_evict", [x] * 5)
