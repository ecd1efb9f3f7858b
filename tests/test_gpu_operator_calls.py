"""How the rotary, account and eviction operators are called: the native path
and the wrappers' own give the same results and errors, on the caller's stream,
from two streams at once and captured into graphs."""

from __future__ import annotations

import pytest
import torch

from cf_hip import layout as L
from cf_hip import ops
from kernels.kv_eviction import evict_move, evict_select
from kernels.paged_attention import chunk_attention_weights, paged_attention_weights
from kernels.rotary import rotary, rotary_cache_write

pytestmark = pytest.mark.gpu


class _None:
    """A native path that takes no call."""

    def __getattr__(self, name):
        return lambda *a: None


class Inputs:
    def __init__(self, gpu, kv, seed=5):
        g = torch.Generator(device=gpu).manual_seed(seed)
        nb, self.h, self.d = 40, 2, 64
        self.kc, self.vc = L.alloc_kv_cache(nb, 16, self.h, self.d, kv, gpu, "paired")
        self.ks = self.vs = None
        if kv == torch.float8_e4m3fn:
            self.ks, self.vs = (torch.tensor(x, device=gpu) for x in ([0.02, 0.03], [0.03, 0.02]))
        rand = lambda *n: torch.randn(*n, generator=g, device=gpu).to(torch.bfloat16)  # noqa: E731
        ops.paged_write(rand(nb * 16, self.h, self.d), torch.arange(nb * 16, device=gpu), self.kc, self.ks)
        ops.paged_write(rand(nb * 16, self.h, self.d), torch.arange(nb * 16, device=gpu), self.vc, self.vs)
        self.q, self.k, self.v = rand(3, 4, self.d), rand(3, self.h, self.d), rand(3, self.h, self.d)
        self.tables = torch.arange(36, dtype=torch.int32, device=gpu).view(3, 12)
        self.lens = torch.tensor([5, 100, 192], dtype=torch.int32, device=gpu)
        self.start = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=gpu)
        self.slots = torch.tensor([7, -1, 300], device=gpu)
        self.pos = torch.tensor([[4, 99, 191], [4, 99, 7], [4, 99, 9]], device=gpu)
        self.freq = torch.rand(32, generator=g, device=gpu)
        self.w = torch.rand(3, self.h, 192, generator=g, device=gpu)
        self.seen = self.lens * 2
        self.kept = torch.tensor([5, 64, 64], dtype=torch.int32, device=gpu)
        self.at = torch.argsort(torch.rand(3, self.h, 192, generator=g, device=gpu), -1).to(torch.int32)

    def state(self):
        raw = [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (self.kc, self.vc)]
        return {"k": raw[0], "v": raw[1], "w": self.w, "at": self.at}

    def all_calls(self):
        """One step of everything, in the order a server has it."""
        out = {"turned": rotary(self.q, self.pos, self.freq, sections=(16, 8, 8), interleaved=True)}
        out["q"] = rotary_cache_write(self.q, self.k, self.v, self.pos, self.freq, self.slots, self.kc, self.vc,
                                      sections=[12, 10, 10], axis_order="cycled", k_scale=self.ks, v_scale=self.vs)
        out["o"] = paged_attention_weights(out["q"], self.kc, self.vc, self.tables, self.lens, self.w, decay=0.5,
                                           k_scale=self.ks, v_scale=self.vs)
        chunk_attention_weights(out["q"], self.kc, self.tables, self.lens, self.start, self.w, observe=1,
                                k_scale=self.ks)
        out["keep"], out["n"] = evict_select(self.w, self.lens, 64, sink=2, recent=8, positions=self.at, kept=self.kept,
                                             seen=self.seen)
        evict_move(out["keep"], self.lens, self.tables, self.kc, self.vc, weights=self.w, positions=self.at,
                   kept=self.kept, seen=self.seen)
        return {**out, **{n: t.clone() for n, t in self.state().items()}}


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float8_e4m3fn])
def test_native_path_equals_the_wrappers_own(gpu, monkeypatch, kv):
    got = Inputs(gpu, kv).all_calls()
    side = torch.cuda.Stream(device=gpu)
    other = Inputs(gpu, kv)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        there = other.all_calls()
    torch.cuda.synchronize()
    monkeypatch.setattr(ops, "_FAST", _None())
    want = Inputs(gpu, kv).all_calls()
    for name in want:
        assert torch.equal(got[name], want[name]) and torch.equal(there[name], want[name]), name


def test_errors_are_the_same_on_both_paths(gpu, monkeypatch):
    x = Inputs(gpu, torch.bfloat16)
    f8 = x.kc.to(torch.float8_e4m3fn)
    bad = [
        lambda: rotary(x.q, x.pos, x.freq),
        lambda: rotary(x.q, x.pos, x.freq, sections=(1, 2)),
        lambda: rotary(x.q, x.pos, x.freq, sections=(16, 8, 9)),
        lambda: rotary(x.q, x.pos, x.freq, sections=(16, 8, 8), axis_order="spiral"),
        lambda: rotary(x.q, x.pos.float(), x.freq, sections=(16, 8, 8)),
        lambda: rotary(x.q, x.pos.cpu(), x.freq, sections=(16, 8, 8)),
        lambda: rotary(x.q.double(), x.pos, x.freq, sections=(16, 8, 8)),
        lambda: rotary(x.q, x.pos, x.freq, sections=(16, 8, 8), out=x.q.float()),
        lambda: rotary_cache_write(x.q, x.k, x.v.float(), x.pos[0], x.freq, x.slots, x.kc, x.vc),
        lambda: rotary_cache_write(x.q, x.k, x.v, x.pos[0], x.freq, x.slots[:2], x.kc, x.vc),
        lambda: rotary_cache_write(x.q, x.k, x.v, x.pos[0], x.freq, x.slots, f8, f8),
        lambda: paged_attention_weights(x.q, x.kc, x.vc, x.tables, x.lens, x.w[:, :, :100]),
        lambda: paged_attention_weights(x.q, x.kc, x.vc, x.tables, x.lens, x.w, 8),
        lambda: paged_attention_weights(x.q, x.kc, x.vc, x.tables, x.lens, x.w, workspace=x.w[0, 0, :64]),
        lambda: paged_attention_weights(x.q, x.kc, x.vc, x.tables, x.lens, x.w, workspace=torch.empty(1 << 24)),
        lambda: paged_attention_weights(x.q[0], x.kc, x.vc, x.tables, x.lens, x.w),
        lambda: chunk_attention_weights(x.q.float(), x.kc, x.tables, x.lens, x.start, x.w),
        lambda: chunk_attention_weights(x.q, x.kc, x.tables, x.lens, x.start, x.w, observe=-1),
        lambda: chunk_attention_weights(x.q, x.kc, x.tables, x.lens, x.start, x.w, observe=1 << 40),
        lambda: chunk_attention_weights(x.q, x.kc, x.tables, x.lens, x.start, x.w, workspace=x.w[0, 0, :64]),
        lambda: evict_select(x.w, x.lens, 0),
        lambda: evict_select(x.w, x.lens, 1 << 31),
        lambda: evict_select(x.w, x.lens, 8, sink=4, recent=5),
        lambda: evict_select(x.w, x.lens, 8, positions=x.at),
        lambda: evict_select(x.w[0], x.lens, 8),
        lambda: evict_select(x.w, x.lens, 8, keep=x.at),
        lambda: evict_move(x.at, x.lens, x.tables, x.kc, x.vc.float()),
        lambda: evict_move(x.at, x.lens, x.tables.cpu(), x.kc, x.vc),
    ]

    def kinds():
        out = []
        for f in bad:
            with pytest.raises(Exception) as e:
                f()
            out.append((e.type, str(e.value)))
        return out

    got = kinds()
    monkeypatch.setattr(ops, "_FAST", _None())
    assert got == kinds()


def test_two_streams_at_once(gpu):
    """Each with a workspace of its own, over caches of its own."""
    a, b = Inputs(gpu, torch.bfloat16, 6), Inputs(gpu, torch.bfloat16, 7)
    want = [Inputs(gpu, torch.bfloat16, 6).all_calls(), Inputs(gpu, torch.bfloat16, 7).all_calls()]
    streams = [torch.cuda.Stream(device=gpu) for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for s, x in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append(x.all_calls())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for name in w:
            assert torch.equal(g[name], w[name]), name


def test_two_graphs_of_the_whole_step(gpu):
    """Two captured steps with workspaces of their own, replayed in turn between eager steps."""
    xs = [Inputs(gpu, torch.float8_e4m3fn, 8 + i) for i in range(2)]
    eager = [Inputs(gpu, torch.float8_e4m3fn, 8 + i) for i in range(2)]
    n1 = ops.decode_weights_workspace_bytes(3, 4, 2, 64, 12, 16)
    n2 = ops.chunk_weights_workspace_bytes(3, 3, 4, 2, 64, 12)
    ws = [(ops.new_workspace(n1, gpu), ops.new_workspace(n2, gpu)) for _ in xs]

    def step(x, ws, out):
        rotary_cache_write(x.q, x.k, x.v, x.pos, x.freq, x.slots, x.kc, x.vc, sections=(12, 10, 10), k_scale=x.ks,
                           v_scale=x.vs, out=out["q"])
        paged_attention_weights(out["q"], x.kc, x.vc, x.tables, x.lens, x.w, k_scale=x.ks, v_scale=x.vs, out=out["o"],
                                workspace=ws[0])
        chunk_attention_weights(out["q"], x.kc, x.tables, x.lens, x.start, x.w, k_scale=x.ks, workspace=ws[1])
        evict_select(x.w, x.lens, 64, sink=2, recent=8, positions=x.at, kept=x.kept, seen=x.seen, keep=out["keep"],
                     new_lens=out["n"])
        evict_move(out["keep"], x.lens, x.tables, x.kc, x.vc, weights=x.w, positions=x.at, kept=x.kept, seen=x.seen)

    def outputs(x):
        return {"q": torch.empty_like(x.q), "o": torch.empty_like(x.q), "n": torch.empty_like(x.lens),
                "keep": torch.empty(3, 2, 64, dtype=torch.int32, device=gpu)}

    warm = Inputs(gpu, torch.float8_e4m3fn, 99)
    step(warm, ws[0], outputs(warm))
    outs, graphs = [outputs(x) for x in xs], []
    torch.cuda.synchronize()
    for x, w, o in zip(xs, ws, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(x, w, o)
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1):
            want = outputs(eager[i])
            xs[i].q.copy_(eager[i].q.mul_(1.1))
            graphs[i].replay()
            step(eager[i], (None, None), want)
            torch.cuda.synchronize()
            for name in want:
                assert torch.equal(outs[i][name], want[name]), (turn, i, name)
            for (name, t), u in zip(xs[i].state().items(), eager[i].state().values()):
                assert torch.equal(t, u), (turn, i, name)


def test_captured_calls_have_workspaces_of_their_own(gpu):
    """Two graphs captured without workspaces, replayed side by side, after a
    larger eager call has replaced the cached ones."""
    xs = [Inputs(gpu, torch.bfloat16, 20 + i) for i in range(2)]
    eager = [Inputs(gpu, torch.bfloat16, 20 + i) for i in range(2)]

    def step(x, out):
        paged_attention_weights(x.q, x.kc, x.vc, x.tables, x.lens, x.w, out=out)
        chunk_attention_weights(x.q, x.kc, x.tables, x.lens, x.start, x.w)

    step(Inputs(gpu, torch.bfloat16, 99), torch.empty_like(xs[0].q))
    outs, graphs = [torch.empty_like(x.q) for x in xs], []
    torch.cuda.synchronize()
    for x, o in zip(xs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(x, o)
        graphs.append(graph)
    big = Inputs(gpu, torch.bfloat16, 30)
    wide = torch.zeros(3, 400, dtype=torch.int32, device=gpu)
    paged_attention_weights(big.q, big.kc, big.vc, wide, big.lens, torch.zeros(3, 2, 6400, device=gpu))
    chunk_attention_weights(big.q, big.kc, wide, big.lens, big.start, torch.zeros(3, 2, 6400, device=gpu))
    streams = [torch.cuda.Stream(device=gpu) for _ in xs]
    for turn in range(4):
        want = [torch.empty_like(o) for o in outs]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for x, e, o, w in zip(xs, eager, outs, want):
            step(e, w)
            assert torch.equal(o, w) and torch.equal(x.w, e.w), turn


def test_int64_tables_and_lengths_are_taken(gpu):
    x, y = Inputs(gpu, torch.bfloat16), Inputs(gpu, torch.bfloat16)
    a = paged_attention_weights(x.q, x.kc, x.vc, x.tables, x.lens, x.w)
    b = paged_attention_weights(y.q, y.kc, y.vc, y.tables.long(), y.lens.long(), y.w)
    assert torch.equal(a, b) and torch.equal(x.w, y.w)
    chunk_attention_weights(x.q, x.kc, x.tables, x.lens, x.start, x.w)
    chunk_attention_weights(y.q, y.kc, y.tables.long(), y.lens.long(), y.start.long(), y.w)
    assert torch.equal(x.w, y.w)
