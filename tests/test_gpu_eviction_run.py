"""A serving run with rotary positions, accounts and evictions through the block
pool, the slabs and the backend, followed by a plain one in float64.

The plain run holds each head's tokens as lists (position, key, value, account).
Keys are checked against the float64 rotary when they are written (half a step
of the stored type, and 3.9e-7 < 2^-21 of the pair's size for the angle, its
sine and cosine and the float32 products, as in tests/test_gpu_rotary.py; an
e4m3fn code's division by its scale rounds once more) and then taken as stored.  Accounts: every weight is within 1.9e-5 of itself
(tests/test_gpu_chunk_weights.py), all terms are positive, and each of the run's
steps rounds the sum twice (decay and addition): 2^-23 a step."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from compiler.cache_policy import CachePolicy
from gpu_util import assert_close
from kernels.kv_eviction import evict_move, evict_select
from kernels.paged_attention import chunk_attention_weights, paged_attention_weights
from kernels.rotary import rotary, rotary_cache_write
from oracle import kv_eviction as plain_evict
from oracle import rotary as plain_rotary
from python_runtime.engine import CacheManager
from python_runtime.engine.block_manager import BlockManager
from python_runtime.hal.hip_backend import HipBackend

pytestmark = pytest.mark.gpu

LAYERS, HKV, G, D, BS, ROWS, COLS = 2, 2, 4, 64, 16, 4, 8
BUDGET, SINK, RECENT, DECAY = 40, 2, 8, 0.96875


class Run:
    def __init__(self, gpu, kv):
        self.gpu, self.kv = gpu, kv
        name = {torch.bfloat16: "bfloat16", torch.float8_e4m3fn: "float8_e4m3fn"}[kv]
        self.mgr = CacheManager(CachePolicy.for_llama(LAYERS, HKV, D, kv_dtype=name), num_blocks=40, device=gpu)
        self.fp8 = kv == torch.float8_e4m3fn
        if self.fp8:
            self.mgr.set_kv_scales("k", torch.tensor([[0.02, 0.03], [0.025, 0.02]]))
            self.mgr.set_kv_scales("v", torch.tensor([[0.03, 0.02], [0.02, 0.025]]))
        self.bm = BlockManager(40, BS)
        self.bm.bind_device(ROWS, COLS, gpu)
        s = COLS * BS
        self.w = torch.full((LAYERS, ROWS, HKV, s), 7.0, device=gpu)  # what is there before a token has no say
        self.at = torch.full((LAYERS, ROWS, HKV, s), -9, dtype=torch.int32, device=gpu)
        self.kept = torch.zeros(ROWS, dtype=torch.int32, device=gpu)
        self.seen = torch.zeros(ROWS, dtype=torch.int32, device=gpu)
        self.freq = (10000.0 ** -(torch.arange(D // 2) / (D // 2))).to(torch.float32).to(gpu)
        self.gen = torch.Generator().manual_seed(11)
        self.tokens: dict[tuple, list] = {}  # (layer, request, head) -> [position, key, value, account]
        self.len: dict[str, int] = {}
        self.pos: dict[str, int] = {}
        self.steps = 0

    def stored(self, slab, layer, slots):
        """Rows at slots as float64 [T, heads, D]."""
        view = self.mgr.layer_view(slab, layer)
        raw = view.view(torch.uint8) if self.fp8 else view
        x = raw[slots // BS, slots % BS]
        if not self.fp8:
            return x.double().cpu().numpy()
        return (x.view(self.kv).float().double() * self.mgr.kv_scales(slab)[layer].double()[:, None]).cpu().numpy()

    def forward(self, counts):
        """Writes counts[r] new tokens of each request and attends with them."""
        rids = list(counts)
        slots, copies = self.bm.prepare_writes([(r, self.len[r], counts[r]) for r in rids])
        BlockManager.copy_blocks(copies, self.mgr.paged_slabs())
        slots = torch.from_numpy(slots).to(self.gpu)
        tables, lens = self.bm.sync_device()
        total = sum(counts.values())
        where = np.concatenate([self.pos[r] + np.arange(counts[r]) for r in rids])
        for r in rids:
            self.seen[self.bm.row_of(r)] += counts[r]
        row = torch.tensor([self.bm.row_of(r) for r in rids], device=self.gpu)
        self.steps += 1
        for layer in range(LAYERS):
            q, k, v = (torch.randn(total, n, D, generator=self.gen).to(torch.bfloat16) for n in (HKV * G, HKV, HKV))
            turned = self.mgr.write_rotary(q.to(self.gpu), k.to(self.gpu), v.to(self.gpu),
                                           torch.from_numpy(where).to(self.gpu), self.freq, slots, layer)
            want, size = plain_rotary.rotate(q.double().numpy(), [where], self.freq.cpu().numpy(), (D // 2,))
            tq = turned.double().cpu().numpy()
            assert (abs(tq - want) <= abs(want) * 2.0**-8 + size * 2.0**-21).all()
            want, size = plain_rotary.rotate(k.double().numpy(), [where], self.freq.cpu().numpy(), (D // 2,))
            ks, vs = self.stored("k", layer, slots), self.stored("v", layer, slots)
            step = 2.0**-4 if self.fp8 else 2.0**-8
            low = 0.03 * 2.0**-10 if self.fp8 else 0.0  # half the smallest e4m3fn step, times the scale
            assert (abs(ks - want) <= abs(want) * step + size * 2.0**-20 + low).all()
            assert (abs(vs - v.double().numpy()) <= abs(v.double().numpy()) * step * (1 + 2.0**-20) + low).all()
            decode = all(n == 1 for n in counts.values())
            if decode:
                qs = torch.zeros(ROWS, HKV * G, D, dtype=torch.bfloat16, device=self.gpu)
                qs[row] = turned
                live = torch.zeros(ROWS, dtype=torch.int32, device=self.gpu)
                live[row] = lens[row]
                out = self.mgr.attend_rows(qs, layer, tables, live, weights=self.w[layer], decay=DECAY)[row]
            else:
                start = torch.tensor(np.cumsum([0, *counts.values()]), dtype=torch.int32, device=self.gpu)
                sub = self.w[layer][row]
                out = self.mgr.attend_chunks(turned, layer, tables[row], lens[row], start, weights=sub, decay=DECAY)
                self.w[layer][row] = sub
            self.follow(layer, counts, where, tq, ks, vs, out.double().cpu().numpy())
        for r in rids:
            self.len[r] += counts[r]
            self.pos[r] += counts[r]

    def follow(self, layer, counts, where, q, k, v, out):
        """The same step in float64, and what it must agree in."""
        want, t = np.zeros_like(out), 0
        for r, n in counts.items():
            for h in range(HKV):
                toks = self.tokens.setdefault((layer, r, h), [])
                old = len(toks)
                for e in toks:
                    e[3] *= DECAY
                for i in range(t, t + n):
                    toks.append([int(where[i]), k[i, h], v[i, h], 0.0])
                for i in range(n):
                    seen = toks[: old + i + 1]
                    kk, vv = np.array([e[1] for e in seen]), np.array([e[2] for e in seen])
                    for j in range(h * G, (h + 1) * G):
                        s = kk @ q[t + i, j] / math.sqrt(D)
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        want[t + i, j] = p @ vv
                        for e, x in zip(seen, p):
                            e[3] += x
                got = self.w[layer, self.bm.row_of(r), h, : old + n].double().cpu().numpy()
                exact = np.array([e[3] for e in toks])
                assert (abs(got - exact) <= exact * (1.9e-5 + self.steps * 2.0**-23)).all()
            t += n
        assert_close(out, want, torch.bfloat16, f"layer {layer}")

    def evict(self):
        """Cuts every request over the budget, in the order the pool's users have it."""
        over = [r for r in self.len if self.len[r] > BUDGET]
        _, copies = self.bm.prepare_writes([(r, 0, BUDGET) for r in over])
        BlockManager.copy_blocks(copies, self.mgr.paged_slabs())
        tables, lens = self.bm.sync_device()
        weights = self.w.double().cpu().numpy()
        for layer in range(LAYERS):
            new = self.mgr.evict_rows(layer, self.w[layer], tables, lens, BUDGET, sink=SINK, recent=RECENT,
                                      positions=self.at[layer], kept=self.kept, seen=self.seen)
        assert new.tolist() == lens.clamp(max=BUDGET).tolist()
        self.kept.copy_(new)
        for r in self.len:
            row, n = self.bm.row_of(r), self.len[r]
            for layer in range(LAYERS):
                for h in range(HKV):
                    toks = self.tokens[(layer, r, h)]
                    pos = np.array([e[0] for e in toks])
                    keep, m = plain_evict.select(weights[layer, row, h], n, BUDGET, SINK, RECENT, pos, n, self.pos[r])
                    self.tokens[(layer, r, h)] = [toks[s] for s in keep[:m]]
            self.len[r] = min(n, BUDGET)
            self.bm.truncate(r, self.len[r])
        self.check()
        return copies

    def check(self):
        """Every request's cache, account and positions are the plain run's."""
        for r, n in self.len.items():
            row, blocks = self.bm.row_of(r), np.array(self.bm.get_blocks(r))
            assert len(blocks) == -(-n // BS)
            t = np.arange(n)
            slots = torch.from_numpy(blocks[t // BS] * BS + t % BS).to(self.gpu)
            for layer in range(LAYERS):
                ks, vs = self.stored("k", layer, slots), self.stored("v", layer, slots)
                for h in range(HKV):
                    toks = self.tokens[(layer, r, h)]
                    assert len(toks) == n
                    assert np.array_equal(ks[:, h], np.array([e[1] for e in toks]))
                    assert np.array_equal(vs[:, h], np.array([e[2] for e in toks]))
                    assert self.at[layer, row, h, :n].tolist() == [e[0] for e in toks]
                    got = self.w[layer, row, h, :n].double().cpu().numpy()
                    exact = np.array([e[3] for e in toks])
                    assert (abs(got - exact) <= exact * (1.9e-5 + self.steps * 2.0**-23)).all()

    def open(self, rid):
        self.bm.allocate(rid, 0)
        self.len[rid] = self.pos[rid] = 0

    def fork(self, src, rid, n):
        """rid starts from src's first n tokens, in the same blocks."""
        self.bm.share_prefix(src, rid, n)
        self.bm.set_len(rid, n)
        self.bm.sync_device()
        a, b = self.bm.row_of(src), self.bm.row_of(rid)
        self.w[:, b] = self.w[:, a]
        self.kept[b], self.seen[b] = 0, n
        self.len[rid] = self.pos[rid] = n
        for (layer, r, h), toks in list(self.tokens.items()):
            if r == src:
                self.tokens[(layer, rid, h)] = [list(e) for e in toks[:n]]


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float8_e4m3fn])
def test_prompts_steps_and_evictions(gpu, kv):
    x = Run(gpu, kv)
    x.open("a")
    x.open("c")
    x.forward({"a": 20, "c": 50})
    x.fork("a", "b", 20)
    x.forward({"b": 12, "a": 1, "c": 3})  # b and a part ways inside a shared block
    x.evict()                             # c alone is over the budget
    x.forward({"c": 20, "b": 25})         # a prompt goes on after an eviction
    copies = x.evict()
    assert len(copies) == 1               # b's first block was still a's too
    for _ in range(3):
        for _ in range(9):
            x.forward({"a": 1, "b": 1, "c": 1})
        x.evict()
    x.bm.free("a")
    del x.len["a"]
    for _ in range(5):
        x.forward({"c": 1, "b": 1})
    x.evict()
    x.bm.free("b")
    x.bm.free("c")
    assert x.bm.num_free_blocks() == 40


def test_backend_ops_are_the_functions(gpu):
    be, g = HipBackend(), torch.Generator(device=gpu).manual_seed(3)

    def inputs():
        g.manual_seed(3)
        rand = lambda *n: torch.randn(*n, generator=g, device=gpu).to(torch.bfloat16)  # noqa: E731
        kc, vc = rand(20, 16, 2, 64), rand(20, 16, 2, 64)
        tables = torch.arange(20, dtype=torch.int32, device=gpu).view(2, 10)
        lens = torch.tensor([33, 150], dtype=torch.int32, device=gpu)
        w = torch.rand(2, 2, 160, generator=g, device=gpu)
        return rand(2, 8, 64), rand(2, 2, 64), rand(2, 2, 64), kc, vc, tables, lens, w

    where = torch.tensor([[32, 149], [0, 2], [0, 5]], device=gpu)
    freq = torch.rand(30, device=gpu)
    slots = torch.tensor([32, 160 + 149], device=gpu)
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    turn = dict(sections=(10, 10, 10), axis_order="cycled", interleaved=True, rotary_scale=1.25)
    at = torch.stack([torch.randperm(160, device=gpu, dtype=torch.int32) for _ in range(4)]).view(2, 2, 160)
    kept, seen = torch.tensor([0, 64], dtype=torch.int32, device=gpu), torch.tensor([33, 400], dtype=torch.int32,
                                                                                  device=gpu)

    def direct():
        q, k, v, kc, vc, tables, lens, w = inputs()
        res = [rotary(q, where, freq, **turn)]
        res.append(rotary_cache_write(q, k, v, where, freq, slots, kc, vc, **turn))
        res.append(paged_attention_weights(res[-1], kc, vc, tables, lens, w, 16, 0.2, decay=0.5))
        res.append(chunk_attention_weights(q, kc, tables, lens, start, w, 16, 0.2, observe=1).clone())
        a = at.clone()
        keep, n = evict_select(w, lens, 48, sink=1, recent=3, positions=a, kept=kept, seen=seen)
        evict_move(keep, lens, tables, kc, vc, weights=w, positions=a, kept=kept, seen=seen)
        return [*res, n, kc, vc, w, a]

    def through():
        q, k, v, kc, vc, tables, lens, w = inputs()
        res = [be.execute("rotary", [q, where, freq], **turn)]
        res.append(be.execute("rotary_cache_write", [q, k, v, where, freq, slots, kc, vc], **turn))
        res.append(be.execute("paged_attention_weights", [res[-1], kc, vc, tables, lens, w], scale=0.2, decay=0.5))
        res.append(be.execute("chunk_attention_weights", [q, kc, tables, lens, start, w], scale=0.2, observe=1).clone())
        a = at.clone()
        n = be.execute("cache_evict", [w, lens, tables, kc, vc, a, kept, seen], budget=48, sink=1, recent=3)
        return [*res, n, kc, vc, w, a]

    for got, want in zip(through(), direct()):
        assert torch.equal(got, want)
    with pytest.raises(ValueError, match="go together"):
        _, _, _, kc, vc, tables, lens, w = inputs()
        be.execute("cache_evict", [w, lens, tables, kc, vc, at], budget=48)
