"""Block-scaled slabs through a serving run: prompts in chunks, decode steps, forks and compactions, followed in
float64 over what the slabs hold."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from block_scaled_util import assert_attended, attend_ref
from compiler.cache_policy import CachePolicy
from python_runtime.engine.block_manager import BlockManager, RequestBatch
from python_runtime.engine.cache.radix_cache import RadixCache
from python_runtime.engine.cache_manager import CacheManager
from python_runtime.hal.hip_backend import HipBackend

pytestmark = pytest.mark.gpu

L, H, HQ, D, BS = 2, 2, 8, 128, 16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _manager(kind, blocks=64):
    return CacheManager(CachePolicy.for_llama(L, H, D), blocks, "cuda", block_scaled=kind)


class Run:
    """The rows every request was given, beside the framework's own state."""

    def __init__(self, kind, rows=8):
        self.mgr, self.bm = _manager(kind), BlockManager(64, BS)
        self.bm.bind_device(rows, 16)
        self.gen = torch.Generator().manual_seed(0)
        self.text = {}  # request -> per layer (k, v) float32 rows [n, H, D]
        self.step = 0

    def rows(self, n):
        return (torch.randn(n, H, D, generator=self.gen) * torch.exp2(torch.randn(n, H, 1, generator=self.gen))).bfloat16()

    def write(self, new):
        """new: {request: rows}; returns the tables, lengths and starts of a step in which each has that many."""
        starts = {r: len(self.text[r][0][0]) if r in self.text else 0 for r in new}
        _, copies = self.bm.prepare_writes_batch(RequestBatch(new), np.array([starts[r] for r in new]),
                                                 np.array(list(new.values())))
        BlockManager.copy_blocks(copies, self.mgr.paged_slabs())
        tables, lens = self.bm.sync_device()
        by_row = sorted(new, key=self.bm.row_of)
        at = [self.bm.row_of(r) for r in by_row]
        counts = [0] * tables.shape[0]
        for r, i in zip(by_row, at):
            counts[i] = new[r]
        start = _i32(np.concatenate([[0], np.cumsum(counts)]).tolist())
        for layer in range(L):
            k, v = self.rows(sum(counts)), self.rows(sum(counts))
            self.mgr.write_rows(k.cuda(), v.cuda(), layer, tables, lens, start)
            i = 0
            for r in by_row:
                had = self.text.setdefault(r, [(torch.empty(0, H, D), torch.empty(0, H, D)) for _ in range(L)])
                had[layer] = tuple(torch.cat([a, b[i: i + new[r]].float()]) for a, b in zip(had[layer], (k, v)))
                i += new[r]
        return tables, lens, start, by_row, at

    def refs(self, layer, request, q, n):
        codes = [self.mgr.layer_view(s, layer).cpu() for s in "kv"]
        scales = [self.mgr.block_scales(s)[:, layer].cpu() for s in "kv"]
        return attend_ref(q, codes[0], scales[0], codes[1], scales[1], self.bm.get_blocks(request), n, D**-0.5)

    def check_values(self, request, kind):
        """What the slabs hold of a request's rows, against the rows themselves."""
        n = len(self.text[request][0][0])
        table = self.bm.get_blocks(request)
        for layer in range(L):
            for s, want in zip("kv", self.text[request][layer]):
                view, sc = self.mgr.layer_view(s, layer).cpu(), self.mgr.block_scales(s)[:, layer].cpu()
                ids = torch.tensor([table[t // BS] for t in range(n)])
                got = view[ids, torch.arange(n) % BS].float() * sc[ids][..., None]
                # a row is rounded once, and int8 ones again at each wider scale, at most 15 times
                tol = 2.0**-4 * want.abs() + 2.0**-9 * sc[ids][..., None] if kind == "float8_e4m3fn" else 8.0 * sc[ids][..., None]
                assert bool(((got - want).abs() <= tol).all())
                # most of them were rounded once or twice
                rms = float((got - want).square().mean().sqrt() / want.square().mean().sqrt())
                assert rms < (0.04 if kind == "float8_e4m3fn" else 0.02)

    def decode(self, requests):
        tables, lens, _, by_row, at = self.write({r: 1 for r in requests})
        for layer in range(L):
            q = torch.randn(tables.shape[0], HQ, D, generator=self.gen).bfloat16()
            live = torch.zeros(tables.shape[0], dtype=torch.int32)
            live[at] = 1
            out = self.mgr.attend_rows(q.cuda(), layer, tables, lens * live.cuda(), self.bm.shared_prefix_lens())
            refs = [self.refs(layer, r, q[i], len(self.text[r][0][0])) for r, i in zip(by_row, at)]
            assert_attended(out[at], refs, torch.bfloat16, D, 250, 2.0**-16, f"decode step {self.step} layer {layer}")
            rest = [i for i in range(tables.shape[0]) if i not in at]
            assert not bool(out[rest].any())
        self.step += 1

    def prefill(self, new):
        tables, lens, start, by_row, at = self.write(new)
        for layer in range(L):
            q = torch.randn(sum(new.values()), HQ, D, generator=self.gen).bfloat16()
            out = self.mgr.attend_chunks(q.cuda(), layer, tables, lens, start)
            pick, refs = [], []
            for r, i in zip(by_row, at):
                n, first = len(self.text[r][0][0]), int(start[i])
                for k in sorted({0, new[r] // 2, new[r] - 1}):
                    pick.append(first + k)
                    refs.append(self.refs(layer, r, q[first + k], n - new[r] + k + 1))
            assert_attended(out[pick], refs, torch.bfloat16, D, 250, 2.0**-11 + 2.0**-16, f"prefill layer {layer}", 2.0**-25)

    def fork(self, src, new_ids):
        copies = self.bm.fork(src, new_ids, len(self.text[src][0][0]))
        BlockManager.move_blocks(copies, self.mgr.paged_slabs())
        for r in new_ids:
            self.text[r] = list(self.text[src])

    def compact(self):
        moves = self.bm.compact()
        BlockManager.move_blocks(moves, self.mgr.paged_slabs())
        self.bm.sync_device()
        return moves


@pytest.mark.parametrize("kind", ["float8_e4m3fn", "int8"])
def test_run(kind):
    run = Run(kind)
    run.prefill({"a": 37, "b": 100, "c": 5})
    for _ in range(3):
        run.decode(["a", "b", "c"])
    run.prefill({"b": 21, "d": 60})  # a chunk that goes on inside a block, and a new prompt
    run.fork("b", ["b1", "b2"])
    run.decode(["a", "b", "b1", "b2", "d"])
    run.bm.free("c")
    run.bm.free("a")
    moves = run.compact()
    assert len(moves) > 0
    for r in ("b", "b1", "b2", "d"):
        run.check_values(r, kind)
    for _ in range(3):
        run.decode(["b", "b1", "b2", "d"])
    run.bm.truncate("d", 50)  # rejected tokens: the next rows go on inside the block
    run.text["d"] = [tuple(x[:50] for x in kv) for kv in run.text["d"]]
    run.prefill({"d": 9, "e": 16})
    run.decode(["b1", "d", "e"])
    for r in ("b", "b1", "b2", "d", "e"):
        run.check_values(r, kind)


def test_shared_prefix_is_copied_before_it_is_written():
    """Copy-on-write takes the scales along: a request that goes on inside a shared block leaves the others'."""
    run = Run("int8")
    run.prefill({"a": 24})
    run.bm.share_prefix("a", "s", 24)
    run.text["s"] = list(run.text["a"])
    was = [run.mgr.layer_view("k", 1).cpu()[run.bm.get_blocks("a")], run.mgr.block_scales("k").cpu()[run.bm.get_blocks("a")]]
    run.write({"s": 4})
    assert torch.equal(run.mgr.layer_view("k", 1).cpu()[run.bm.get_blocks("a")], was[0])
    assert torch.equal(run.mgr.block_scales("k").cpu()[run.bm.get_blocks("a")], was[1])
    assert run.bm.get_blocks("a")[0] == run.bm.get_blocks("s")[0] and run.bm.get_blocks("a")[1] != run.bm.get_blocks("s")[1]
    run.check_values("s", "int8")
    run.check_values("a", "int8")


def test_radix_cache_follows_a_compaction():
    run = Run("float8_e4m3fn")
    run.prefill({"x": 20, "a": 48, "y": 3})
    radix = RadixCache(run.bm)
    text = list(range(100, 148))
    radix.insert(text, run.bm.get_blocks("a"))
    run.bm.free("x")
    radix.relocate(run.compact())
    blocks, matched = radix.match_prefix(text + [1])
    assert matched == 48 and blocks == run.bm.get_blocks("a")
    run.check_values("a", "float8_e4m3fn")


@pytest.mark.parametrize("kind", ["float8_e4m3fn", "int8"])
def test_reads_and_attend(kind):
    """read_paged and attend, the manager's methods over host tables."""
    mgr = _manager(kind, 12)
    gen = torch.Generator().manual_seed(3)
    tables = {"b": [4, 2, 9], "a": [7, 1]}
    k, v = (torch.randn(60, H, D, generator=gen).bfloat16() for _ in range(2))
    mgr.begin_step(tables)
    mgr.write_rows(k.cuda(), v.cuda(), 1, _i32([[7, 1, -1], [4, 2, 9]]), _i32([20, 40]), _i32([0, 20, 60]))
    got = mgr.read_paged("k", 1, 40).cpu()
    assert got.dtype == torch.float32 and got.shape == (2, 40, H, D)
    step = 2.0**-4 if kind == "float8_e4m3fn" else 0.0
    scale = mgr.block_scales("k")[:, 1].cpu()
    assert bool(((got[1] - k[20:].float()).abs() <= step * k[20:].float().abs() + 0.5001 * scale.max()).all())
    q = torch.randn(2, HQ, D, generator=gen).bfloat16()
    out = mgr.attend(q.cuda(), 1, [20, 40])
    codes = [mgr.layer_view(s, 1).cpu() for s in "kv"]
    sc = [mgr.block_scales(s)[:, 1].cpu() for s in "kv"]
    refs = [attend_ref(q[i], codes[0], sc[0], codes[1], sc[1], t, n, D**-0.5) for i, (t, n) in enumerate((([7, 1], 20), ([4, 2, 9], 40)))]
    assert_attended(out, refs, torch.bfloat16, D, 40, 2.0**-16, "attend")


def test_what_block_scaled_slabs_refuse():
    mgr = _manager("int8", 8)
    rows, slots = torch.zeros(2, H, D, dtype=torch.bfloat16, device="cuda"), torch.tensor([0, 1])
    t, n = _i32([[0], [1]]), _i32([1, 1])
    q = torch.zeros(2, HQ, D, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2, H, 16, device="cuda")
    mgr.begin_step({"a": [0], "b": [1]})
    with pytest.raises(NotImplementedError):
        mgr.write_slots("k", 0, rows, slots)
    with pytest.raises(NotImplementedError):
        mgr.write_paged("k", 0, rows, torch.tensor([0, 1]))
    with pytest.raises(NotImplementedError):
        mgr.write_rotary(q, rows, rows, n, torch.ones(4, device="cuda"), slots, 0)
    with pytest.raises(NotImplementedError):
        mgr.attend_rows(q, 0, t, n, weights=w)
    with pytest.raises(NotImplementedError):
        mgr.attend_chunks(q, 0, t, n, _i32([0, 1, 2]), weights=w)
    with pytest.raises(NotImplementedError):
        mgr.evict_rows(0, w, t, n, 8)
    with pytest.raises(ValueError):
        mgr.kv_scales("k")
    with pytest.raises(ValueError):
        mgr.set_kv_scales("k", torch.ones(L, H))
    plain = CacheManager(CachePolicy.for_llama(L, H, D, kv_dtype="float8_e4m3fn"), 8, "cuda")
    with pytest.raises(ValueError, match="not block-scaled"):
        plain.write_rows(rows, rows, 0, t, n)
    with pytest.raises(ValueError, match="no block scales"):
        plain.block_scales("k")
    assert len(mgr.paged_slabs()) == 4 and len(plain.paged_slabs()) == 2


def test_backend_ops():
    """The HAL's ops over a block-scaled cache."""
    mgr = _manager("int8", 8)
    hal = HipBackend()
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(20, H, D, generator=gen).bfloat16().cuda() for _ in range(2))
    kc, vc = mgr.layer_view("k", 0), mgr.layer_view("v", 0)
    ks, vs = mgr.block_scales("k")[:, 0], mgr.block_scales("v")[:, 0]
    t, n, start = _i32([[3, 5]]), _i32([20]), _i32([0, 20])
    assert hal.execute("kv_cache_write_blocks", [k, v, t, n, kc, vc, ks, vs, start]) is kc
    both = hal.execute("cache_read", [kc, vc, t], seq_len=20, k_scale=ks, v_scale=vs)
    assert both.dtype == torch.float32
    assert float((both[0, 0] - k.float()).norm() / k.float().norm()) < 0.02
    q = torch.randn(20, HQ, D, generator=gen).bfloat16().cuda()
    rows = hal.execute("chunked_prefill_attention", [q, kc, vc, t, n, start], k_scale=ks, v_scale=vs)
    last = hal.execute("paged_attention", [q[19:], kc, vc, t, n], k_scale=ks, v_scale=vs)
    assert float((rows[19].double() - last[0].double()).norm() / last.double().norm()) < 2.0**-7
    with pytest.raises(ValueError):
        hal.execute("kv_cache_write_blocks", [k, v, t, n])
