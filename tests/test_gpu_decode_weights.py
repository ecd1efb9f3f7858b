"""Decode attention with accounts on the GPU: the output is the plain call's,
the accounts those of the softmax in float64.

Tolerance of a weight p = exp(s - m) / l in float32: the score s (log2 units,
|s| <= 16 here) is a sum of D products rounded to |s| * 2^-24 a step of a short
tree, at worst 2^-21 of sum |q k| in all, and scaled with one rounding (2^-24 *
16); a change of s by e changes p by p * e * ln 2; exp2 and the division add 3
ulp, l its own sum's 2^-20.  Together, with scores of |q||k| * scale <= 16:
below 1.2e-5 * p; an account adds at most 16 of them and its old value, half a
step each."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from cf_hip import layout as L
from cf_hip import ops
from kernels.paged_attention import paged_attention_tensors, paged_attention_weights

pytestmark = pytest.mark.gpu
REL = 1.2e-5


class Case:
    def __init__(self, gpu, b, hq, h, d, lens, q_dtype, kv, layout="paired", bs=16, seed=0, mb=None, hw=None, peak=1.0):
        g = torch.Generator(device=gpu).manual_seed(seed)
        self.lens, self.bs = lens, bs
        mb = mb or max(1, -(-max(lens) // bs))
        nb = b * mb + 5
        self.tables = torch.randperm(nb, generator=torch.Generator().manual_seed(seed))[: b * mb].view(b, mb).to(
            torch.int32).to(gpu)
        self.k, self.v = (self._odd if layout == "odd" else L.alloc_kv_cache)(nb, bs, h, d, kv, gpu, layout)
        self.ks = self.vs = None
        for i, c in enumerate((self.k, self.v)):
            x = torch.randn(nb, bs, h, d, generator=g, device=gpu)
            if kv == torch.float8_e4m3fn:
                sc = 0.016 + 0.004 * torch.rand(h, generator=g, device=gpu)
                c.view(torch.uint8).copy_((x / sc[:, None]).to(kv).view(torch.uint8))
                self.ks, self.vs = (sc, None) if i == 0 else (self.ks, sc)
            else:
                c.copy_(x.to(kv))
        self.q = (torch.randn(b, hq, d, generator=g, device=gpu) * peak).to(q_dtype)
        self.seq = torch.tensor(lens, dtype=torch.int32, device=gpu)
        self.w = torch.rand(b, h if hw is None else hw, mb * bs, generator=g, device=gpu)
        self.scale = 1.0 / math.sqrt(d)

    @staticmethod
    def _odd(nb, bs, h, d, dtype, gpu, _):
        return tuple(torch.zeros(bs, h, nb, 2 * d, dtype=dtype, device=gpu)[..., ::2].permute(2, 0, 1, 3)
                     for _ in range(2))

    def run(self, **more):
        return paged_attention_weights(self.q, self.k, self.v, self.tables, self.seq, self.w, self.bs, k_scale=self.ks,
                                       v_scale=self.vs, **more)

    def plain(self, **more):
        return paged_attention_tensors(self.q, self.k, self.v, self.tables, self.seq, self.bs, k_scale=self.ks,
                                       v_scale=self.vs, **more)

    def rows(self, cache, scale, b, h):
        n = min(max(self.lens[b], 0), self.tables.shape[1] * self.bs)
        t = torch.arange(n, device=cache.device)
        blk = self.tables[b][t // self.bs].long()
        ok = (blk >= 0) & (blk < cache.shape[0])
        raw = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
        x = raw[blk.clamp(0, cache.shape[0] - 1), t % self.bs, h]
        x = x.view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else x
        x = x.float().double()
        return (x if scale is None else x * scale[h].double()), ok

    def weights(self):
        """[B, Hq, S] softmax weights in float64."""
        b, hq, _ = self.q.shape
        h = self.k.shape[2]
        out = torch.zeros(b, hq, self.w.shape[2], dtype=torch.float64, device=self.q.device)
        for i in range(b):
            for j in range(hq):
                k, ok = self.rows(self.k, self.ks, i, j // (hq // h))
                if bool(ok.any()):
                    s = torch.where(ok, k @ self.q[i, j].double() * self.scale, -math.inf)
                    out[i, j, : len(s)] = torch.softmax(s, 0)
        return out

    def expected(self, before, decay):
        p = self.weights()
        b, hq, s = p.shape
        add = p.view(b, self.w.shape[1], -1, s).sum(2)
        want = before.double().clone()
        for i, n in enumerate(self.lens):
            m = min(max(n, 0), self.tables.shape[1] * self.bs)
            old = want[i, :, :m] * decay if decay else torch.zeros_like(want[i, :, :m])
            if 0 < n <= m:
                old[:, n - 1] = 0.0
            want[i, :, :m] = old + add[i, :, :m]
        return want, add


def _check(case, decay=1.0, **more):
    before = case.w.clone()
    want, add = case.expected(before, decay)
    out = case.run(decay=decay, **more)
    got = case.w.double()
    err = (got - want).abs()
    bound = add * (REL + 2.0**-22) + want.abs() * 2.0**-22 + 1e-37
    assert bool((err <= bound).all()), float((err / bound).max())
    same = case.plain(**more)
    assert torch.equal(out, same)
    return out


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float8_e4m3fn), (torch.float16, torch.float16),
         (torch.float16, torch.float8_e4m3fn), (torch.float32, torch.float32), (torch.float32, torch.bfloat16),
         (torch.float32, torch.float8_e4m3fn)]


@pytest.mark.parametrize("q, kv", TYPES)
@pytest.mark.parametrize("layout", ["paired", "native", "token_major"])
@pytest.mark.parametrize("hq, h, d", [(4, 4, 64), (8, 1, 64), (32, 8, 128), (32, 2, 128)])
def test_types_and_heads(gpu, q, kv, layout, hq, h, d):
    _check(Case(gpu, 4, hq, h, d, [1, 33, 511, 700], q, kv, layout, seed=1))


@pytest.mark.parametrize("q, kv", [(torch.float32, torch.float32), (torch.bfloat16, torch.float16),
                                   (torch.float16, torch.float8_e4m3fn), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("hq, h, d, bs", [(6, 2, 40, 16), (3, 3, 80, 8), (5, 1, 256, 1), (8, 8, 64, 32)])
@pytest.mark.parametrize("layout", ["token_major", "odd"])
def test_other_shapes(gpu, q, kv, hq, h, d, bs, layout):
    _check(Case(gpu, 3, hq, h, d, [1, 70, 600], q, kv, layout, bs, seed=2))


@pytest.mark.parametrize("decay", [1.0, 0.5, 0.0, -1.0])
@pytest.mark.parametrize("hw", [None, 1])
def test_decay_and_one_account(gpu, decay, hw):
    case = Case(gpu, 3, 16, 4, 64, [40, 1, 257], torch.bfloat16, torch.bfloat16, seed=3, hw=hw)
    case.w[:, :, 39::7] = float("nan") if decay == 0.0 else 0.5
    if decay != 0.0:  # the newest tokens' entries are not read either
        for i, n in enumerate(case.lens):
            case.w[i, :, n - 1] = float("nan")
    before = case.w.clone()
    want, add = case.expected(before.nan_to_num(0.0), decay)
    case.run(decay=decay)
    for i, n in enumerate(case.lens):
        err = (case.w[i, :, :n].double() - want[i, :, :n]).abs()
        assert bool((err <= add[i, :, :n] * (REL + 2.0**-22) + want[i, :, :n].abs() * 2.0**-22).all())
        assert torch.equal(case.w[i, :, n:].nan_to_num(9.0), before[i, :, n:].nan_to_num(9.0))


@pytest.mark.parametrize("q, kv", [(torch.bfloat16, torch.float8_e4m3fn), (torch.float32, torch.float32)])
@pytest.mark.parametrize("b, n", [(1, 20000), (2, 9001), (300, 40)])
def test_long_and_many(gpu, q, kv, b, n):
    _check(Case(gpu, b, 8, 2, 128, [max(1, n - 3 * i) for i in range(b)], q, kv, seed=4))


def test_more_sequences_than_a_plan_holds(gpu):
    _check(Case(gpu, 2100, 2, 1, 64, [1 + i % 37 for i in range(2100)], torch.bfloat16, torch.bfloat16, seed=5))


@pytest.mark.parametrize("d, hq, h", [(128, 32, 8), (64, 4, 4)])
def test_shared_prefixes(gpu, d, hq, h):
    """Sharers of one prefix, each with an account of its own; one sequence ends inside the shared part."""
    case = Case(gpu, 6, hq, h, d, [300, 290, 160, 500, 64, 200], torch.bfloat16, torch.float8_e4m3fn, seed=6)
    case.tables[1:4, :10] = case.tables[0, :10]
    shared = torch.tensor(ops.shared_prefix_lens(case.tables.tolist(), case.lens, 16), dtype=torch.int32, device=gpu)
    assert shared.tolist()[1:4] == [160, 160, 160]
    _check(case, shared_prefix_lens=shared)


def test_accounts_in_a_launch_of_their_own(gpu):
    """Tables so wide that the rows are joined first: a shared prefix, and the partitioned kernel."""
    case = Case(gpu, 6, 16, 4, 64, [300, 290, 160, 0, 64, 5000], torch.bfloat16, torch.float8_e4m3fn, seed=12, mb=2800)
    case.tables[1:3, :10] = case.tables[0, :10]
    shared = torch.tensor([0, 160, 160, 0, 0, 0], dtype=torch.int32, device=gpu)
    _check(case, shared_prefix_lens=shared)
    _check(Case(gpu, 3, 6, 2, 40, [1000, 1, 3000], torch.float32, torch.float32, "token_major", seed=13, mb=11000))


def test_many_partitions(gpu):
    _check(Case(gpu, 1, 6, 2, 40, [40000], torch.float32, torch.bfloat16, "token_major", seed=14))


def test_lengths_at_the_edges_and_invalid_blocks(gpu):
    case = Case(gpu, 6, 8, 2, 64, [0, -3, 48, 90, 33, 48], torch.bfloat16, torch.bfloat16, seed=7, mb=3)
    case.tables[4, 1] = -1
    case.tables[5, :] = case.k.shape[0]  # nothing to attend to
    out = _check(case)
    assert bool((out[[0, 1, 5]] == 0).all())


def test_invalid_blocks_on_the_partitioned_kernel(gpu):
    case = Case(gpu, 3, 6, 2, 40, [48, 90, 1], torch.float32, torch.float32, "token_major", seed=8, mb=3)
    case.tables[0, 1], case.tables[2, 0] = -1, 1 << 30
    _check(case)


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float32])
def test_nan_scores_reach_their_own_row_only(gpu, kv):
    case = Case(gpu, 2, 8, 2, 64, [50, 50], torch.float32 if kv == torch.float32 else kv, kv, seed=9)
    case.k[case.tables[0, 1].item(), 3, 1] = float("nan")
    clean = Case(gpu, 2, 8, 2, 64, [50, 50], torch.float32 if kv == torch.float32 else kv, kv, seed=9)
    case.run()
    clean.run()
    assert bool(case.w[0, 1, :50].isnan().all())
    assert torch.equal(case.w[0, 0], clean.w[0, 0]) and torch.equal(case.w[1], clean.w[1])


def test_a_peaked_softmax(gpu):
    case = Case(gpu, 2, 8, 2, 128, [1000, 333], torch.bfloat16, torch.bfloat16, seed=10)
    case.q *= 12
    before = case.w.clone()
    want, _ = case.expected(before, 1.0)
    case.run()
    # scores up to 12 times as large, and their errors with them
    err = (case.w.double() - want).abs()
    assert bool((err <= (want - before).abs() * 12 * REL + want * 2.0**-22).all())


def test_strided_accounts_and_a_workspace(gpu):
    case = Case(gpu, 2, 8, 2, 64, [100, 77], torch.bfloat16, torch.bfloat16, seed=11)
    big = torch.zeros(2, 3, 2, 150, device=gpu)
    case.w = big[:, 1, :, 3:131]  # rows apart, not 16-byte aligned
    need = ops.decode_weights_workspace_bytes(2, 8, 2, 64, case.tables.shape[1], 16)
    _check_rest = big.clone()
    out = torch.empty_like(case.q)
    want, add = case.expected(case.w, 1.0)
    got = case.run(out=out, workspace=ops.new_workspace(need, gpu))
    assert got is out
    assert bool(((case.w.double() - want).abs() <= add * REL + want * 2.0**-22).all())
    _check_rest[:, 1, :, 3:131] = case.w
    assert torch.equal(big, _check_rest)
    with pytest.raises(ValueError, match="workspace"):
        case.run(workspace=ops.new_workspace(need, gpu)[: need - 1])


def test_repeats_are_equal(gpu):
    a, b = (Case(gpu, 5, 32, 8, 128, [900, 20, 3000, 511, 64], torch.bfloat16, torch.float8_e4m3fn, seed=12)
            for _ in range(2))
    for _ in range(3):
        assert torch.equal(a.run(), b.run())
    assert torch.equal(a.w, b.w)


def test_capture_and_replay(gpu):
    """A captured call with its own workspace, replayed between eager calls."""
    cap, eager = (Case(gpu, 4, 32, 8, 128, [900, 20, 3000, 511], torch.bfloat16, torch.float8_e4m3fn, seed=13)
                  for _ in range(2))
    need = ops.decode_weights_workspace_bytes(4, 32, 8, 128, cap.tables.shape[1], 16)
    ws, out = ops.new_workspace(need, gpu), torch.empty_like(cap.q)
    cap.run(out=out, workspace=ws)  # (loads the kernels)
    eager.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap.run(out=out, workspace=ws)
    for i in range(4):
        cap.q.copy_(eager.q.mul_(0.9))
        out.zero_()
        graph.replay()
        want = eager.run()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(cap.w, eager.w), i


@pytest.mark.parametrize("hw", [None, 1])
@pytest.mark.parametrize("q, kv", [(torch.bfloat16, torch.float8_e4m3fn), (torch.float32, torch.float32)])
def test_tables_and_accounts_much_wider_than_the_sequences(gpu, q, kv, hw):
    """The engine's own tables: 2,048 columns for sequences of a few blocks, rows without a request among them."""
    case = Case(gpu, 5, 8, 2, 64, [40, 0, 1, 511, 200], q, kv, seed=31, hw=hw)
    tables = torch.full((5, 2048), -1, dtype=torch.int32, device=gpu)
    w = torch.rand(5, case.w.shape[1], 2048 * 16 + 3, device=gpu)
    for i, m in enumerate(case.lens):
        tables[i, : -(-m // 16)] = case.tables[i, : -(-m // 16)]
    case.tables, case.w = tables, w
    rest = w.clone()
    _check(case, decay=0.5)
    for i, m in enumerate(case.lens):
        assert torch.equal(w[i, :, m:], rest[i, :, m:])
