"""Accounts of prompt chunks on the GPU against the softmax in float64.

Tolerance: a weight p is within 1.2e-5 p of the exact one for log2 scores up to
16 (tests/test_gpu_decode_weights.py has the terms); an account adds them in
float32, four a step of a workgroup's stretch (84 in a chain at most here), then
16 lanes in four steps and the runs in five, half a step each: 93 * 2^-24 =
5.6e-6 of the sum; l is a sum of 35 roundings at most, 1.2e-6 more than the
2^-20 counted there: below 7e-6 together, and a step of the whole for the old
value."""

from __future__ import annotations

import math

import pytest
import torch

from cf_hip import layout as L
from cf_hip import ops
from kernels.paged_attention import chunk_attention_weights, paged_attention_weights

pytestmark = pytest.mark.gpu
REL = 1.2e-5 + 7e-6


class Case:
    def __init__(self, gpu, chunks, hq, h, d, q_dtype, kv, layout="paired", seed=0, hw=None, mb=None, gaps=0):
        """chunks: (rows, cached tokens) each; gaps: rows of q between chunks' that belong to none."""
        g = torch.Generator(device=gpu).manual_seed(seed)
        self.chunks = chunks
        self.lens = [r + c for r, c in chunks]
        mb = mb or max(1, -(-max(self.lens) // 16))
        nb = len(chunks) * mb + 5
        self.tables = torch.randperm(nb, generator=torch.Generator().manual_seed(seed))[: len(chunks) * mb].view(
            len(chunks), mb).to(torch.int32).to(gpu)
        self.k, v = L.alloc_kv_cache(nb, 16, h, d, kv, gpu, layout)
        x = torch.randn(nb, 16, h, d, generator=g, device=gpu)
        self.ks = None
        if kv == torch.float8_e4m3fn:
            self.ks = 0.016 + 0.004 * torch.rand(h, generator=g, device=gpu)
            self.k.view(torch.uint8).copy_((x / self.ks[:, None]).to(kv).view(torch.uint8))
        else:
            self.k.copy_(x.to(kv))
        self.starts = [gaps]
        for r, _ in chunks:
            self.starts.append(self.starts[-1] + r)
        self.start = torch.tensor(self.starts, dtype=torch.int32, device=gpu)
        self.q = torch.randn(self.starts[-1] + gaps, hq, d, generator=g, device=gpu).to(q_dtype)
        self.seq = torch.tensor(self.lens, dtype=torch.int32, device=gpu)
        self.w = torch.rand(len(chunks), h if hw is None else hw, mb * 16, generator=g, device=gpu)
        self.scale = 1.0 / math.sqrt(d)

    def run(self, **more):
        return chunk_attention_weights(self.q, self.k, self.tables, self.seq, self.start, self.w, k_scale=self.ks,
                                       **more)

    def expected(self, decay=1.0, observe=0, scale=None):
        scale = self.scale if scale is None else scale
        hq, h = self.q.shape[1], self.k.shape[2]
        hw, cap = self.w.shape[1], self.tables.shape[1] * 16
        want = self.w.double().clone()
        add = torch.zeros_like(want)
        for n, n_tok in enumerate(self.lens):
            a, b = self.starts[n], self.starts[n + 1]
            if b <= a or n_tok <= 0:
                continue
            m = min(n_tok, cap)
            t = torch.arange(m, device=self.q.device)
            blk = self.tables[n][t // 16].long()
            ok = (blk >= 0) & (blk < self.k.shape[0])
            rows = torch.arange(max(a, b - observe) if observe else a, b, device=self.q.device)
            pos = n_tok - b + rows
            sees = ok[None] & (t[None] <= pos[:, None])
            for j in range(hq):
                hk = j // (hq // h)
                raw = self.k.view(torch.uint8) if self.ks is not None else self.k
                x = raw[blk.clamp(0, self.k.shape[0] - 1), t % 16, hk]
                x = x.view(self.k.dtype).float().double() * self.ks[hk].double() if self.ks is not None else x.double()
                s = (x @ self.q[rows, j].double().T.contiguous()).T * scale
                p = torch.softmax(torch.where(sees, s, -math.inf), 1)
                p = torch.where(sees.any(1, keepdim=True), p, 0.0)
                add[n, hk if hw > 1 else 0, :m] += p.sum(0)
            old = want[n, :, :m] * decay if decay else torch.zeros_like(want[n, :, :m])
            old[:, max(0, n_tok - (b - a)):] = 0.0
            want[n, :, :m] = old + add[n, :, :m]
        return want, add


def _check(case, **more):
    want, add = case.expected(**more)
    got = case.run(**more)
    assert got is case.w
    err = (case.w.double() - want).abs()
    bound = add * REL + want.abs() * 2.0**-23 + 1e-37
    assert bool((err <= bound).all()), (float((err / bound).max()), int((err > bound).sum()))


# blocks of the tables: as many as the tokens take, and the widths at which four
# waves, eight, or kernels for rows and tokens apart take them
WIDTHS = pytest.mark.parametrize("mb", [None, 24, 40])
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float8_e4m3fn), (torch.float16, torch.float16),
         (torch.float16, torch.float8_e4m3fn)]


@pytest.mark.parametrize("q, kv", TYPES)
@pytest.mark.parametrize("layout", ["paired", "native", "token_major"])
@pytest.mark.parametrize("hq, h, d", [(4, 4, 64), (8, 1, 64), (32, 8, 128), (16, 1, 128)])
@pytest.mark.parametrize("mb, most", [(None, 150), (None, 300), (40, 300)])
def test_types_and_heads(gpu, q, kv, layout, hq, h, d, mb, most):
    _check(Case(gpu, [(1, 0), (17, 30), (130, 0), (64, most)], hq, h, d, q, kv, layout, seed=1, mb=mb))


@pytest.mark.parametrize("hq, h", [(6, 2), (3, 1), (64, 1), (20, 4), (1, 1)])
@WIDTHS
def test_groups_that_are_no_power_of_two(gpu, hq, h, mb):
    _check(Case(gpu, [(100, 45), (7, 0)], hq, h, 64, torch.bfloat16, torch.bfloat16, seed=2, mb=mb))


@pytest.mark.parametrize("rows, cached", [(1, 0), (1, 999), (15, 1), (16, 16), (255, 1), (256, 0), (257, 255), (1000, 24),
                                          (2100, 0), (3, 5000)])
def test_one_chunk(gpu, rows, cached):
    _check(Case(gpu, [(rows, cached)], 8, 2, 64, torch.bfloat16, torch.bfloat16, seed=3))


@pytest.mark.parametrize("observe", [1, 2, 16, 64, 1000])
@pytest.mark.parametrize("hw", [None, 1])
def test_observers(gpu, observe, hw):
    _check(Case(gpu, [(90, 700), (20, 3), (1, 0), (300, 0)], 16, 4, 128, torch.bfloat16, torch.float8_e4m3fn, seed=4,
                hw=hw), observe=observe)


@pytest.mark.parametrize("decay", [0.0, 0.5, -2.0])
@pytest.mark.parametrize("hw", [None, 1])
@WIDTHS
def test_decay(gpu, decay, hw, mb):
    case = Case(gpu, [(33, 64), (5, 100)], 8, 4, 64, torch.float16, torch.float16, seed=5, hw=hw, mb=mb)
    want, add = case.expected(decay=decay)
    for n, (r, c) in enumerate(case.chunks):  # entries without history are not read
        case.w[n, :, c: r + c] = float("nan")
        if decay == 0.0:
            case.w[n, :, :c] = float("nan")
    rest = case.w.clone()
    case.run(decay=decay)
    for n, m in enumerate(case.lens):
        err = (case.w[n, :, :m].double() - want[n, :, :m]).abs()
        assert bool((err <= add[n, :, :m] * REL + want[n, :, :m].abs() * 2.0**-23).all())
        assert torch.equal(case.w[n, :, m:], rest[n, :, m:])


def test_large_units_and_many_pieces(gpu):
    """Enough rows for the wide units, long enough for several pieces of tokens."""
    _check(Case(gpu, [(2500, 0), (1024, 2000), (2000, 70)], 32, 8, 64, torch.bfloat16, torch.bfloat16, seed=6))


@WIDTHS
def test_many_chunks(gpu, mb):
    _check(Case(gpu, [(1 + i % 5, i * 7 % 90) for i in range(270)], 4, 2, 64, torch.bfloat16, torch.bfloat16, seed=7,
                gaps=3, mb=mb))


@WIDTHS
def test_chunks_without_rows_and_odd_starts(gpu, mb):
    case = Case(gpu, [(10, 20), (0, 50), (30, 0), (5, 5)], 8, 2, 64, torch.bfloat16, torch.bfloat16, seed=8, mb=mb)
    before = case.w[1].clone()
    _check(case)
    assert torch.equal(case.w[1], before)
    # a start before the previous chunk's end starts there; ends past q are cut
    case = Case(gpu, [(10, 20), (6, 50), (24, 10)], 8, 2, 64, torch.bfloat16, torch.bfloat16, seed=9, mb=mb)
    case.start = torch.tensor([0, 10, 4, 999], dtype=torch.int32, device=gpu)
    case.starts = [0, 10, 10, 40]
    case.lens = [30, 56, 34]
    _check(case)


@pytest.mark.parametrize("mb", [3, 24, 40])
def test_lengths_at_the_edges_and_invalid_blocks(gpu, mb):
    case = Case(gpu, [(40, 8), (20, 0), (20, 28), (48, 0), (48, 0)], 8, 2, 64, torch.bfloat16, torch.bfloat16, seed=10,
                mb=mb)
    case.lens = [mb * 16 + 52, 7, 0, 48, 48]  # past the table, shorter than the chunk, empty
    case.seq = torch.tensor(case.lens, dtype=torch.int32, device=gpu)
    case.tables[3, 1] = -1
    case.tables[4, :] = case.k.shape[0]
    _check(case)


@WIDTHS
def test_nan_scores_stay_in_their_rows(gpu, mb):
    bad, clean = (Case(gpu, [(64, 0), (64, 0)], 8, 2, 64, torch.bfloat16, torch.bfloat16, seed=11, mb=mb)
                  for _ in range(2))
    bad.q[20, 1] = float("nan")  # chunk 0, KV head 0
    bad.run()
    clean.run()
    assert bool(bad.w[0, 0, :21].isnan().all()) and torch.equal(bad.w[0, 0, 21:], clean.w[0, 0, 21:])
    assert torch.equal(bad.w[0, 1], clean.w[0, 1]) and torch.equal(bad.w[1], clean.w[1])


@pytest.mark.parametrize("kv", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [64, 70, 83])  # x 4 heads: whole steps of columns, and not
@WIDTHS
def test_infinite_keys_that_no_row_attends_to(gpu, kv, rows, mb):
    """A key channel of +inf that every query meets with a negative value: its token's score is
    -inf and its weight 0, whatever the last step's columns past the rows hold."""
    case = Case(gpu, [(rows, 200), (9, 0)], 8, 2, 64, kv, kv, seed=16, mb=mb)
    case.q[:, :, 5] = -case.q[:, :, 5].abs() - 0.5
    for t in (10, 130):
        case.k[int(case.tables[0, t // 16]), t % 16, :, 5] = math.inf
    _check(case)


@pytest.mark.parametrize("observe", [0, 16])
@pytest.mark.parametrize("hw", [None, 1])
@pytest.mark.parametrize("chunks", [[(77, 0), (1, 30), (38, 12)], [(500, 0)] * 8, [(40, 1900), (300, 100)]])
def test_tables_and_accounts_much_wider_than_the_sequences(gpu, chunks, hw, observe):
    """The engine's own tables: 2,048 columns for sequences of a few blocks, no block past their end."""
    case = Case(gpu, chunks, 8, 2, 64, torch.bfloat16, torch.bfloat16, seed=17, hw=hw)
    n = len(chunks)
    tables = torch.full((n, 2048), -1, dtype=torch.int32, device=gpu)
    w = torch.rand(n, case.w.shape[1], 2048 * 16 + 5, device=gpu)
    for i, m in enumerate(case.lens):
        tables[i, : -(-m // 16)] = case.tables[i, : -(-m // 16)]
    case.tables, case.w = tables, w
    rest = w.clone()
    _check(case, observe=observe)
    for i, m in enumerate(case.lens):
        assert torch.equal(w[i, :, m:], rest[i, :, m:])


@pytest.mark.parametrize("scale", [-0.125, 0.0])
@WIDTHS
def test_negative_and_zero_scales(gpu, scale, mb):
    case = Case(gpu, [(70, 20), (9, 0)], 8, 2, 64, torch.float16, torch.float8_e4m3fn, seed=12, mb=mb)
    _check(case, scale=scale)


def test_single_rows_agree_with_decode(gpu):
    case = Case(gpu, [(1, 400), (1, 0), (1, 77)], 16, 4, 128, torch.bfloat16, torch.bfloat16, seed=13)
    w = case.w.clone()
    case.run(decay=0.5)
    paged_attention_weights(case.q, case.k, case.k, case.tables, case.seq, w, decay=0.5)
    assert bool(((w - case.w).abs() <= w * 2 * REL).all())


def test_strides_and_a_workspace(gpu):
    case = Case(gpu, [(50, 30), (20, 0)], 8, 2, 64, torch.bfloat16, torch.bfloat16, seed=14)
    big_q = torch.zeros(70, 24, 64, dtype=torch.bfloat16, device=gpu)
    big_q[:, 8:16] = case.q  # the queries of a fused projection
    case.q = big_q[:, 8:16]
    big = torch.rand(2, 3, 2, 99, device=gpu)
    case.w = big[:, 1, :, 3:83]
    rest = big.clone()
    need = ops.chunk_weights_workspace_bytes(70, 2, 8, 2, 64, case.tables.shape[1])
    _check(case, **{})
    rest[:, 1, :, 3:83] = case.w
    assert torch.equal(big, rest)
    case.run(workspace=ops.new_workspace(need, gpu))
    with pytest.raises(ValueError, match="workspace"):
        case.run(workspace=ops.new_workspace(need, gpu)[: need - 1])


def test_what_it_does_not_take(gpu):
    for change in (dict(q_dtype=torch.float32, kv=torch.float32), dict(q_dtype=torch.bfloat16, kv=torch.float16),
                   dict(q_dtype=torch.bfloat16, kv=torch.bfloat16, d=96)):
        a = dict(chunks=[(4, 0)], hq=4, h=2, d=64) | change
        case = Case(gpu, **a)
        with pytest.raises((NotImplementedError, ValueError)):
            case.run()


def test_repeats_and_replays_are_equal(gpu):
    cap, eager = (Case(gpu, [(300, 900), (64, 3000)], 32, 8, 128, torch.bfloat16, torch.float8_e4m3fn, seed=15)
                  for _ in range(2))
    need = ops.chunk_weights_workspace_bytes(364, 2, 32, 8, 128, cap.tables.shape[1])
    ws = ops.new_workspace(need, gpu)
    cap.run(workspace=ws)
    eager.run()
    assert torch.equal(cap.w, eager.w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap.run(workspace=ws, decay=0.5)
    for i in range(4):
        cap.q.copy_(eager.q.mul_(0.9))
        graph.replay()
        eager.run(decay=0.5)
        torch.cuda.synchronize()
        assert torch.equal(cap.w, eager.w), i
