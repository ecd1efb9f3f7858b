"""Block-scaled caches, block moves, fork and compaction: what is refused before any launch, and the host's
bookkeeping (no GPU)."""

from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest
import torch

from cf_hip import _abi, layout, ops
from cf_hip.layout import alloc_kv_cache, alloc_kv_scales
from compiler.cache_policy import CachePolicy
from kernels.block_scaled_kv import write_kv_blocks
from python_runtime.engine.block_manager import BlockManager
from python_runtime.engine.cache.radix_cache import RadixCache
from python_runtime.engine.cache_manager import CacheManager


def _desc(t: torch.Tensor) -> _abi.CfTensor:
    """A descriptor that claims device memory: every check runs, and a refused call launches nothing."""
    d = _abi.descriptor(t)
    d.t.device = _abi.SFA_ROCM
    return d


def _message() -> str:
    return _abi.last_error()


def _write_args(**other):
    a = dict(k_new=torch.zeros(3, 2, 64, dtype=torch.bfloat16), v_new=torch.zeros(3, 2, 64, dtype=torch.bfloat16),
             block_tables=torch.zeros(3, 4, dtype=torch.int32), seq_lens=torch.ones(3, dtype=torch.int32), q_start=None,
             k_cache=torch.zeros(8, 16, 2, 64, dtype=torch.int8), v_cache=torch.zeros(8, 16, 2, 64, dtype=torch.int8),
             k_scale=torch.zeros(8, 2), v_scale=torch.zeros(8, 2))
    a.update(other)
    return a


def _write(**other) -> int:
    d = [_desc(t) if t is not None else None for t in _write_args(**other).values()]
    return _abi.lib().cf_kv_write_blocks(*(_abi.ref(x) for x in d), None)


@pytest.mark.parametrize("other, says", [
    (dict(k_new=torch.zeros(3, 2, 64, dtype=torch.int32)), "k_new: dtype"),
    (dict(v_new=torch.zeros(3, 2, 64, dtype=torch.float16)), "v_new dtype"),
    (dict(v_new=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), "v_new shape"),
    (dict(k_new=torch.zeros(3, 2, 32, dtype=torch.bfloat16), v_new=torch.zeros(3, 2, 32, dtype=torch.bfloat16)), "does not match new rows"),
    (dict(k_cache=torch.zeros(8, 16, 2, 64, dtype=torch.bfloat16)), "k_cache: dtype must be f8e4m3fn or i8"),
    (dict(v_cache=torch.zeros(8, 16, 2, 64, dtype=torch.float8_e4m3fn)), "v_cache dtype"),
    (dict(v_cache=torch.zeros(9, 16, 2, 64, dtype=torch.int8)), "v_cache shape"),
    (dict(k_scale=torch.zeros(2)), "k_scale: expected rank 2"),
    (dict(k_scale=torch.zeros(8, 3)), "k_scale: expected [8, 2]"),
    (dict(v_scale=torch.zeros(8, 2, dtype=torch.float16)), "v_scale: expected f32"),
    (dict(v_scale=torch.zeros(1, 2).expand(8, 2)), "v_scale: rows overlap"),
    (dict(k_cache=torch.zeros(1, 16, 2, 64, dtype=torch.int8).expand(8, 16, 2, 64)), "k_cache: rows overlap"),
    (dict(block_tables=torch.zeros(3, 4, dtype=torch.int64)), "block_tables: expected i32"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int32)), "seq_lens has 2 entries"),
    (dict(q_start=torch.zeros(3, dtype=torch.int32)), "q_start has 3 entries"),
    (dict(q_start=torch.zeros(4, dtype=torch.int64)), "q_start: expected i32"),
    (dict(block_tables=torch.zeros(2, 4, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32)), "3 rows for 2 sequences"),
])
def test_write_refuses(other, says):
    assert _write(**other) == _abi.CF_ERR_INVALID
    assert says in _message()


def test_write_of_nothing_is_no_launch():
    """Empty calls return before any launch: no rows, no blocks, no table columns."""
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16)
    assert _write(k_new=none, v_new=none, block_tables=torch.zeros(0, 4, dtype=torch.int32),
                  seq_lens=torch.zeros(0, dtype=torch.int32)) == 0
    assert _write(block_tables=torch.zeros(3, 0, dtype=torch.int32)) == 0
    empty = torch.zeros(0, 16, 2, 64, dtype=torch.int8)
    assert _write(k_cache=empty, v_cache=empty, k_scale=torch.zeros(0, 2), v_scale=torch.zeros(0, 2)) == 0


def _decode(kv, ks, vs, weights=False) -> int:
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    cache = torch.zeros(8, 16, 2, 64, dtype=kv)
    d = [_desc(t) if t is not None else None
         for t in (q, cache, cache, torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32), None, ks, vs)]
    out = _desc(torch.zeros_like(q))
    if weights:
        w = _desc(torch.zeros(2, 2, 64))
        return _abi.lib().cf_paged_decode_weights(*(_abi.ref(x) for x in d), 0.125, 16, _abi.ref(w), 1.0, _abi.ref(out), None,
                                                  0, None)
    return _abi.lib().cf_paged_decode_shared(*(_abi.ref(x) for x in d), 0.125, 16, 512, _abi.ref(out), None, 0, None)


@pytest.mark.parametrize("kv, ks, vs, says", [
    (torch.int8, torch.ones(2), torch.ones(2), "i8 with block scales"),
    (torch.int8, None, None, "i8 with block scales"),
    (torch.bfloat16, torch.ones(8, 2), torch.ones(8, 2), "block scales apply to"),
    (torch.float8_e4m3fn, torch.ones(8, 2), torch.ones(2), "v_scale: expected rank 2"),
    (torch.float8_e4m3fn, torch.ones(8, 2), None, "v_scale: descriptor is NULL"),
    (torch.float8_e4m3fn, torch.ones(2), torch.ones(8, 2), "v_scale: expected rank 1"),
    (torch.int8, torch.ones(7, 2), torch.ones(8, 2), "k_scale: expected [8, 2]"),
    (torch.int8, torch.ones(8, 2), torch.ones(8, 1), "v_scale: expected [8, 2]"),
    (torch.int8, torch.ones(8, 2, dtype=torch.float16), torch.ones(8, 2), "k_scale: expected f32"),
])
def test_decode_refuses(kv, ks, vs, says):
    assert _decode(kv, ks, vs) == _abi.CF_ERR_INVALID
    assert says in _message()


def test_accounts_are_refused():
    assert _decode(torch.int8, torch.ones(8, 2), torch.ones(8, 2), weights=True) == _abi.CF_ERR_UNSUPPORTED
    assert _decode(torch.float8_e4m3fn, torch.ones(8, 2), torch.ones(8, 2), weights=True) == _abi.CF_ERR_UNSUPPORTED
    assert "accounts" in _message()


@pytest.mark.parametrize("kv, ks, vs, says", [
    (torch.int8, torch.ones(2), torch.ones(2), "i8 with block scales"),
    (torch.bfloat16, torch.ones(8, 2), torch.ones(8, 2), "block scales apply to"),
    (torch.float8_e4m3fn, torch.ones(8, 2), torch.ones(2), "v_scale: expected rank 2"),
    (torch.int8, torch.ones(8, 2), torch.ones(2, 8), "v_scale: expected [8, 2]"),
])
def test_prefill_refuses(kv, ks, vs, says):
    q = torch.zeros(5, 4, 64, dtype=torch.bfloat16)
    cache = torch.zeros(8, 16, 2, 64, dtype=kv)
    d = [_desc(t) for t in (q, cache, cache, torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                            torch.tensor([0, 5], dtype=torch.int32), ks, vs)]
    out = _desc(torch.zeros_like(q))
    rc = _abi.lib().cf_prefill_chunk_fp8(*(_abi.ref(x) for x in d), 0.125, 16, _abi.ref(out), None, 0, None)
    assert rc == _abi.CF_ERR_INVALID
    assert says in _message()


def test_single_row_writers_refuse_int8():
    rows, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    cache = torch.zeros(8, 16, 2, 64, dtype=torch.int8)
    d = [_desc(t) for t in (rows, slots, cache, torch.ones(2))]
    assert _abi.lib().cf_paged_write(*(_abi.ref(x) for x in d), None) == _abi.CF_ERR_INVALID


def _moves(caches, moves) -> int:
    d = (_abi.CfTensor * max(len(caches), 1))(*(_desc(c) for c in caches))
    m = np.asarray(moves, dtype=np.int32).reshape(-1, 2)
    return _abi.lib().cf_move_blocks(d, len(caches), m.ctypes.data, len(m), None)


@pytest.mark.parametrize("moves, says", [
    ([(0, 8)], "outside the caches' 8 blocks"), ([(-1, 2)], "outside"), ([(9, 2)], "outside"),
    ([(0, 2), (1, 3), (4, 2)], "block 2 is the destination of two moves"),
])
def test_moves_refuse(moves, says):
    cache = torch.zeros(8, 40, dtype=torch.uint8)
    assert _moves([cache], moves) == _abi.CF_ERR_INVALID
    assert says in _message()


def test_write_refuses_one_tensor_for_both():
    rows, cache = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 8, 16, 2, 64, dtype=torch.int8)
    scale, one = torch.ones(2, 8, 2), torch.ones(1, dtype=torch.int32)
    for c, s in (((0, 0), (0, 1)), ((0, 1), (1, 1))):
        d = [_desc(t) for t in (rows, rows, torch.zeros(1, 4, dtype=torch.int32), one)]
        d += [None] + [_desc(t) for t in (cache[c[0]], cache[c[1]], scale[s[0]], scale[s[1]])]
        rc = _abi.lib().cf_kv_write_blocks(*(None if x is None else _abi.ref(x) for x in d), None)
        assert rc == _abi.CF_ERR_INVALID and "cannot share" in _message()


def test_write_refuses_more_blocks_than_a_launch_takes():
    row, one = torch.zeros(1, 1, 8, dtype=torch.bfloat16), torch.ones(1, dtype=torch.int32)
    n = 1 << 24
    many = row.expand(n, 1, 8)  # (descriptors only: nothing is read)
    cache, scale = torch.zeros(2, 8, 16, 1, 8, dtype=torch.int8), torch.ones(2, 8, 1)
    d = [_desc(t) for t in (many, many, one.view(1, 1).expand(n, 1), one.expand(n), cache[0], cache[1], scale[0], scale[1])]
    rc = _abi.lib().cf_kv_write_blocks(*(_abi.ref(x) for x in d[:4]), None, *(_abi.ref(x) for x in d[4:]), None)
    assert rc == _abi.CF_ERR_INVALID and "16777216 blocks" in _message()


def test_moves_refuse_a_cache_twice():
    cache = torch.zeros(8, 40, dtype=torch.uint8)
    assert _moves([cache, torch.zeros(8, 4, dtype=torch.uint8), cache], [(1, 7)]) == _abi.CF_ERR_INVALID
    assert "given twice" in _message()


def test_moves_refuse_caches_that_share_memory():
    slab = torch.zeros(8, 3, 40, dtype=torch.uint8)
    flat = torch.zeros(1000, dtype=torch.uint8)
    for caches in ([slab, slab[:, 1]], [slab[:, 2], slab[:, :1], slab[:, 1:]], [slab[:6, 1], slab[4:, 1]],
                   [flat[:320].view(8, 40), flat[300:620].view(8, 40)],
                   [flat[:320].view(8, 40), flat[319:327].view(8, 1)],
                   [flat.as_strided((8, 30), (100, 1), 0), flat.as_strided((3, 30), (100, 1), 729)],
                   [flat.as_strided((8, 30), (100, 1), 0), flat.as_strided((3, 31), (100, 1), 670)],
                   [flat.as_strided((8, 30), (100, 1), 0), flat.as_strided((8, 25), (75, 1), 50)],
                   [flat.as_strided((8, 30), (100, 1), 0), flat.as_strided((7, 50), (100, 1), 90)]):
        flats = [c.as_strided((c.shape[0], c.shape[1:].numel()), (c.stride(0), 1)) for c in caches]
        assert _moves(flats, [(0, 1)]) == _abi.CF_ERR_INVALID
        assert "share memory" in _message()


def test_paired_storage():
    k, v = layout.alloc_kv_cache(6, 16, 2, 8, torch.int8, "cpu", "paired")
    k.copy_(torch.randint(-9, 9, k.shape))
    v.copy_(torch.randint(-9, 9, v.shape))
    both = layout.paired_storage(k, v)
    assert both.is_contiguous() and both.data_ptr() == k.data_ptr() and both.shape == (6, 2, 2, 128)
    assert torch.equal(both[:, :, 0].view(6, 2, 16, 8), k.transpose(1, 2))
    assert torch.equal(both[:, :, 1].view(6, 2, 8, 16), v.permute(0, 2, 3, 1))
    with pytest.raises(ValueError, match="one paired cache"):
        layout.paired_storage(*layout.alloc_kv_cache(6, 16, 2, 8, torch.int8, "cpu", "native"))
    with pytest.raises(ValueError, match="one paired cache"):
        layout.paired_storage(k, layout.alloc_kv_cache(6, 16, 2, 8, torch.int8, "cpu", "paired")[1])


def test_moves_refuse_caches():
    assert _moves([torch.zeros(8, 40, dtype=torch.uint8), torch.zeros(6, 40, dtype=torch.uint8)], [(1, 7)]) == _abi.CF_ERR_INVALID
    assert "6 blocks" in _message()
    assert _moves([torch.zeros(8, 4, 10, dtype=torch.uint8)], [(1, 7)]) == _abi.CF_ERR_INVALID
    assert _moves([torch.zeros(8, 80, dtype=torch.uint8)[:, ::2]], [(1, 7)]) == _abi.CF_ERR_INVALID
    assert _moves([torch.zeros(8, dtype=torch.uint8).as_strided((8, 4), (0, 1))], [(1, 7)]) == _abi.CF_ERR_INVALID
    assert "overlap" in _message()
    assert _moves([], [(1, 7)]) == 0 and _moves([torch.zeros(8, 40, dtype=torch.uint8)], []) == 0


def test_moves_python_refusals():
    cache = torch.zeros(8, 4)
    with pytest.raises(ValueError, match="ROCm device tensor"):
        BlockManager.move_blocks([(0, 1)], [cache])
    for bad in ([(0.5, 1.0)], [(0, 1, 2)], [0, 1], [(-1, 3)], [(0, 1 << 31)]):
        with pytest.raises(ValueError):
            ops.move_blocks([], bad)
    ops.move_blocks([], [])
    ops.move_blocks([], np.empty((0, 2), dtype=np.int64))


def test_python_refusals_without_a_gpu():
    a = {k: v for k, v in _write_args().items() if k != "q_start"}
    with pytest.raises(ValueError, match="ROCm device tensor"):
        write_kv_blocks(**a)
    with pytest.raises(ValueError, match="block_scaled must be"):
        CacheManager(CachePolicy.for_llama(2, 2, 64).to_dict() if hasattr(CachePolicy, "for_llama") else {}, 4, "cpu",
                     block_scaled="int4")


def test_scales_lie_side_by_side():
    k, v = alloc_kv_scales(6, 3, "cpu")
    assert k.shape == v.shape == (6, 3) and k.dtype == torch.float32
    assert v.data_ptr() - k.data_ptr() == 12 and k.stride() == (6, 1)
    assert alloc_kv_cache(2, 16, 3, 64, torch.int8, "cpu")[0].dtype == torch.int8


# ---- fork and compaction ---------------------------------------------------------------


def test_fork_shares_whole_blocks_and_copies_the_last():
    bm = BlockManager(16, 4)
    blocks = bm.allocate("a", 11)
    copies = bm.fork("a", ["b", "c", "d"], 10)
    assert [c[0] for c in copies.tolist()] == [blocks[2]] * 3
    for i, r in enumerate("bcd"):
        assert bm.get_blocks(r) == blocks[:2] + [copies[i, 1]]
    assert len({int(c) for c in copies[:, 1]} | set(blocks)) == 6
    assert bm.ref_count(blocks[0]) == 4 and bm.ref_count(blocks[2]) == 1
    assert bm.num_allocated_blocks() == 6
    assert len(bm.prepare_writes([("b", 10, 1), ("c", 10, 1)])[1]) == 0  # nothing is shared any more
    for r in "abcd":
        bm.free(r)
    assert bm.num_free_blocks() == 16


def test_fork_at_a_block_boundary_copies_nothing():
    bm = BlockManager(8, 4)
    blocks = bm.allocate("a", 8)
    assert bm.fork("a", ["b"], 8).shape == (0, 2) and bm.get_blocks("b") == blocks
    assert bm.fork("a", ["c"], 0).shape == (0, 2) and bm.get_blocks("c") == []
    assert bm.fork("a", [], 7).shape == (0, 2)


def test_fork_refuses_and_changes_nothing():
    bm = BlockManager(6, 4)
    bm.allocate("a", 6)
    bm.allocate("x", 4)
    free = bm.num_free_blocks()
    with pytest.raises(KeyError):
        bm.fork("none", ["b"], 4)
    for ids, tokens in ((["b"], 9), (["b", "b"], 6), (["b", "x"], 6), (["a"], 6), (["b"], -1)):
        with pytest.raises(ValueError):
            bm.fork("a", ids, tokens)
    with pytest.raises(RuntimeError):
        bm.fork("a", ["b", "c", "d", "e"], 6)  # three blocks are free
    assert bm.num_free_blocks() == free and bm.ref_count(bm.get_blocks("a")[0]) == 1
    with pytest.raises(KeyError):
        bm.get_blocks("b")


def test_fork_reaches_the_device_rows():
    bm = BlockManager(16, 4)
    bm.bind_rows(4, 8)
    bm.prepare_writes([("a", 0, 10)])
    bm.table_deltas()
    bm.fork("a", ["b"], 10)
    d = bm.table_deltas().tolist()
    row = bm.row_of("b")
    assert sorted(x[2] for x in d if x[0] == row and x[1] >= 0) == sorted(bm.get_blocks("b"))
    assert [x[2] for x in d if x[0] == row and x[1] == -1] == [10]


def test_compact_lays_the_requests_out_in_order():
    rng = random.Random(0)
    bm = BlockManager(64, 4)
    bm.bind_rows(16, 16)
    for i in range(10):
        bm.prepare_writes([(f"r{i}", 0, rng.randint(1, 20))])
    bm.table_deltas()
    for i in (1, 4, 7):
        bm.free(f"r{i}")
    bm.share_prefix("r0", "s", 4)
    rest = [f"r{i}" for i in (0, 2, 3, 5, 6, 8, 9)]
    for r in rest[2:]:
        bm.prepare_writes([(r, 20, 9)])
    radix = RadixCache(bm)
    bm.allocate("p", 8)
    held = bm.get_blocks("p")
    radix.insert(list(range(8)), held)
    bm.free("p")  # only the prefix cache holds them now
    old = {r: bm.get_blocks(r) for r in rest + ["s"]}
    counts = {b: bm.ref_count(b) for t in old.values() for b in t}
    used = bm.num_allocated_blocks()
    moves = bm.compact()
    assert bm.compact().shape == (0, 2)  # in order already (rows are as they were)
    now = dict(moves.tolist())
    assert len(now) == len(moves) and len(set(now.values())) == len(now) and all(a != b for a, b in now.items())
    at = lambda b: now.get(b, b)  # noqa: E731
    for r, t in old.items():
        assert bm.get_blocks(r) == [at(b) for b in t]
        assert [bm.ref_count(at(b)) for b in t] == [counts[b] for b in t]
    flat = [b for r in rest for b in bm.get_blocks(r)]
    assert flat == list(range(len(flat)))  # device rows are in this order
    radix.relocate(moves)
    assert radix.match_prefix(list(range(8))) == ([at(b) for b in held], 8)
    assert sorted(at(b) for b in held) == [used - 2, used - 1]
    assert bm.num_allocated_blocks() == used
    assert bm.allocate("new", 8) == [used, used + 1]  # the pool's end is free, the lowest taken next
    # the device rows follow: what the deltas say, applied to the old rows, is the new tables
    d = bm.table_deltas()
    cells = {(int(r), int(c)): int(v) for r, c, v, _ in d if c >= 0}
    for r in rest:
        row = bm.row_of(r)
        assert [cells.get((row, j), b) for j, b in enumerate(old[r])] == bm.get_blocks(r)


def test_compact_counts_without_a_change():
    bm = BlockManager(8, 4)
    bm.allocate("a", 9)
    n = ctypes.c_int64(0)
    assert _abi.lib().cf_bp_compact(bm._h, None, 0, ctypes.byref(n)) == 0 and n.value == 3
    assert bm.get_blocks("a") == [7, 6, 5]
    buf = np.empty((1, 2), dtype=np.int32)
    assert _abi.lib().cf_bp_compact(bm._h, buf.ctypes.data, 1, ctypes.byref(n)) == _abi.CF_ERR_INVALID
    assert bm.get_blocks("a") == [7, 6, 5]
    assert bm.compact().tolist() == [[5, 2], [6, 1], [7, 0]]
    assert bm.get_blocks("a") == [0, 1, 2]
