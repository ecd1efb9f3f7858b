"""Eviction by accumulated weight on the GPU: the selection against the plain
statement (oracle/kv_eviction.py), the moves against indexing."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cf_hip import layout as L
from cf_hip import ops
from kernels.kv_eviction import evict_move, evict_select
from oracle import kv_eviction as oracle

pytestmark = pytest.mark.gpu


def _weights(gpu, b, h, s, seed, kind):
    g = torch.Generator(device=gpu).manual_seed(seed)
    w = torch.empty(b, h, s, device=gpu).exponential_(generator=g)
    if kind == "ties":
        w = (w * 3).floor()
    elif kind == "odd":  # zeros of both signs, infinities, NaN of both signs, subnormals, negative numbers
        odd = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), -float("nan"), 1e-42, -1e-42, -3.0,
                            3.4e38], device=gpu)
        pick = torch.randint(0, 14, w.shape, generator=g, device=gpu)
        w = torch.where(pick < 10, odd[pick.clamp(max=9)], w)
    elif kind == "equal":
        w.fill_(0.25)
    elif kind == "nan":
        w.fill_(float("nan"))
    return w


def _check_select(w, lens, budget, sink, recent, pos=None, kept=None, seen=None):
    gpu = w.device
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    before = w.clone()
    keep, new = evict_select(w, i32(lens), budget, sink=sink, recent=recent, positions=pos, kept=i32(kept),
                             seen=i32(seen))
    assert torch.equal(w.nan_to_num(7.0), before.nan_to_num(7.0))
    assert keep.dtype == new.dtype == torch.int32 and keep.shape == (*w.shape[:2], budget)
    keep, new, wn = keep.cpu().numpy(), new.tolist(), w.cpu().numpy()
    for b, n in enumerate(lens):
        n = min(max(n, 0), w.shape[2])
        for h in range(w.shape[1]):
            p = None if pos is None else pos[b, h].cpu().numpy()
            want, m = oracle.select(wn[b, h], n, budget, sink, recent, p, 0 if kept is None else kept[b],
                                    n if seen is None else seen[b])
            assert new[b] == m
            assert np.array_equal(keep[b, h], want), (b, h, np.nonzero(keep[b, h] != want)[0][:4])


@pytest.mark.parametrize("kind", ["plain", "ties", "odd", "equal", "nan"])
@pytest.mark.parametrize("s, budget, sink, recent", [
    (1, 1, 0, 0), (16, 1, 0, 1), (64, 63, 4, 8), (1000, 100, 1, 99), (1040, 1024, 4, 64), (4097, 2048, 0, 0),
])
def test_select_small(gpu, kind, s, budget, sink, recent):
    w = _weights(gpu, 3, 2, s, 11, kind)
    _check_select(w, [s, min(s, budget), max(0, s - 7)], budget, sink, recent)


@pytest.mark.parametrize("kind", ["plain", "ties"])
@pytest.mark.parametrize("s, n, budget", [(9000, 8999, 3000), (20001, 20001, 10001), (40000, 33333, 20000),
                                          (70000, 70000, 9000)])
def test_select_long(gpu, kind, s, n, budget):
    """Each register width, the variant without them, and more movers than one hand-over holds."""
    w = _weights(gpu, 1, 2, s, 12, kind)
    _check_select(w, [n], budget, 4, 64)


def test_select_lengths_at_the_edges(gpu):
    w = _weights(gpu, 6, 1, 48, 13, "plain")
    _check_select(w, [0, -5, 1, 32, 33, 1000], 32, 2, 3)  # past the buffer: all of its slots


def test_select_with_positions_and_strides(gpu):
    b, h, s, budget = 3, 2, 200, 90
    g = torch.Generator(device=gpu).manual_seed(3)
    w = _weights(gpu, h, b, 300, 14, "ties").transpose(0, 1)[:, :, 50: 50 + s]  # rows far apart, heads outermost
    kept, lens, seen = [90, 60, 0], [180, 200, 150], [1000, 400, 150]
    pos = torch.full((b, h, s), -7, dtype=torch.int32, device=gpu)  # (unused past kept)
    for i in range(b):
        for j in range(h):
            at = torch.randperm(seen[i] - (lens[i] - kept[i]), generator=g, device=gpu)[: kept[i]]
            pos[i, j, : kept[i]] = at.to(torch.int32)
    _check_select(w, lens, budget, 4, 30, pos, kept, seen)
    _check_select(w, lens, budget, 0, 90, pos, kept, seen)


@pytest.mark.parametrize("kind", ["plain", "ties"])
@pytest.mark.parametrize("s, budget", [(900, 300), (2000, 700), (6000, 2048), (12000, 2500), (30000, 4096), (40000, 9000)])
def test_select_with_positions_at_every_width(gpu, kind, s, budget):
    """Stored positions with each kernel: sequences near their buffer's end and far from it, whose last
    waves hold nothing, some of whose protected tokens lie anywhere in their slots."""
    g = torch.Generator(device=gpu).manual_seed(s)
    h = 2 if s < 10000 else 1
    lens = [s, s - s // 10 - 3, s // 2 + 1, budget + 1]
    kept = [s // 2, budget, s // 3, budget]
    seen = [3 * n for n in lens]
    w = _weights(gpu, len(lens), h, s, 15, kind)
    pos = torch.full((len(lens), h, s), -7, dtype=torch.int32, device=gpu)  # (unused past kept)
    for i in range(len(lens)):
        for j in range(h):
            at = torch.randperm(seen[i] - (lens[i] - kept[i]), generator=g, device=gpu)[: kept[i]]
            pos[i, j, : kept[i]] = at.to(torch.int32)
        # the text's first tokens and some of its latest, wherever they are
        pos[i, :, kept[i] // 3: kept[i] // 3 + 4] = torch.arange(4, dtype=torch.int32, device=gpu)
    _check_select(w, lens, budget, 4, budget // 2, pos, kept, seen)
    _check_select(w, lens, budget, 4, min(budget - 4, s // 20), pos, kept, seen)


@pytest.mark.parametrize("s", [4096, 12000, 32000, 40000])
def test_accounts_much_wider_than_the_sequences(gpu, s):
    """A bounded cache's accounts, as wide as the longest prompt: sequences near the budget, and one
    that has no token."""
    w = _weights(gpu, 5, 2, s, 18, "plain")
    _check_select(w, [2064, 2049, 2048, 17, 0], 2048, 4, 256)


def test_select_takes_columns_of_one_tensor(gpu):
    """Lengths side by side in one tensor, the new ones among them."""
    w = _weights(gpu, 3, 2, 300, 16, "plain")
    state = torch.tensor([[300, 64, 500], [150, 100, 150], [40, 0, 40]], dtype=torch.int32, device=gpu)
    new = torch.zeros(3, 4, dtype=torch.int32, device=gpu)
    new[:, 1:] = state
    pos = torch.arange(300, dtype=torch.int32, device=gpu).expand(3, 2, 300).contiguous()
    want = evict_select(w, state[:, 0], 64, sink=2, recent=9, positions=pos, kept=state[:, 1], seen=state[:, 2])
    got = evict_select(w, new[:, 1], 64, sink=2, recent=9, positions=pos, kept=new[:, 2], seen=new[:, 3],
                       new_lens=new[:, 0])
    assert torch.equal(got[0], want[0]) and torch.equal(new[:, 0], want[1]) and torch.equal(new[:, 1:], state)
    for shared in (1, 2, 3):
        with pytest.raises(ValueError, match="new_lens must not share"):
            evict_select(w, new[:, 1], 64, sink=2, recent=9, positions=pos, kept=new[:, 2], seen=new[:, 3],
                         new_lens=new[:, shared])
    with pytest.raises(ValueError, match="new_lens must not share"):
        evict_select(w, new[:, 1], 64, new_lens=new[:, 1])


def _fill(t, seed):
    g = torch.Generator(device=t.device).manual_seed(seed)
    raw = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]
    info = torch.iinfo(raw)
    t.view(raw).copy_(torch.randint(info.min, info.max, t.shape, generator=g, device=t.device).to(raw))
    return t.view(raw)


def _caches(gpu, nb, bs, h, d, dtype, layout, seed=5):
    if layout == "odd":  # channels apart, tokens outermost
        pair = [torch.zeros(bs, h, nb, 2 * d, dtype=dtype, device=gpu)[..., ::2].permute(2, 0, 1, 3) for _ in range(2)]
    else:
        pair = L.alloc_kv_cache(nb, bs, h, d, dtype, gpu, layout)
    for i, c in enumerate(pair):
        _fill(c, seed + i)
    return pair


def _raw(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def _expected(cache, keep, tables, hw):
    """The cache after the moves, by indexing one row at a time."""
    want = cache.clone()
    bs = cache.shape[1]
    for b in range(keep.shape[0]):
        for h in range(hw):
            heads = slice(None) if hw == 1 else slice(h, h + 1)
            for j, src in enumerate(keep[b, h].tolist()):
                if src >= 0 and src != j:
                    t, f = int(tables[b, j // bs]), int(tables[b, src // bs])
                    if 0 <= t < cache.shape[0] and 0 <= f < cache.shape[0]:
                        want[t, j % bs, heads] = cache[f, src % bs, heads]
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("layout", ["paired", "native", "token_major", "odd"])
@pytest.mark.parametrize("bs, d, hw", [(16, 64, 2), (16, 128, 1), (8, 40, 2), (1, 3, 1)])
def test_move(gpu, dtype, layout, bs, d, hw):
    h, lens, budget = 2, [75, 64, 20, 0, 90], 40
    mb = -(-96 // bs)
    nb = len(lens) * mb + 3
    k, v = _caches(gpu, nb, bs, h, d, dtype, layout)
    w = _weights(gpu, len(lens), hw, mb * bs, 21, "plain")
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    tables = perm[: len(lens) * mb].view(len(lens), mb).to(gpu)
    tables[1, 0] = -1  # no such block: its rows stay
    tables[4, 1] = nb
    tl = torch.tensor(lens, dtype=torch.int32, device=gpu)
    keep, _ = evict_select(w, tl, budget, sink=2, recent=8)
    want = [_expected(_raw(c), keep, tables, hw) for c in (k, v)]
    ww = w.clone()
    for b in range(len(lens)):
        for i in range(hw):
            m = keep[b, i][keep[b, i] >= 0].long()
            ww[b, i, : m.numel()] = w[b, i][m]
    evict_move(keep, tl, tables, k, v, weights=w)
    assert torch.equal(_raw(k), want[0]) and torch.equal(_raw(v), want[1]) and torch.equal(w, ww)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("layout", ["paired", "native", "token_major"])
@pytest.mark.parametrize("bs, d, hw", [(16, 64, 2), (32, 40, 1), (16, 136, 1), (16, 8, 2)])
def test_move_of_many(gpu, dtype, layout, bs, d, hw):
    """Most slots of a sequence move, few of another's, none of a third's; runs
    that end at the budget, and blocks that the cache does not have."""
    h, lens, budget = 2, [1100, 320, 296, 700], 297
    mb = -(-1120 // bs)
    nb = len(lens) * mb + 3
    k, v = _caches(gpu, nb, bs, h, d, dtype, layout)
    w = _weights(gpu, len(lens), hw, mb * bs, 23, "plain")
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(2)).to(torch.int32)
    tables = perm[: len(lens) * mb].view(len(lens), mb).to(gpu)
    tables[0, 1], tables[0, mb // 2], tables[3, mb // 3] = -1, nb, 1 << 30
    tl = torch.tensor(lens, dtype=torch.int32, device=gpu)
    keep, _ = evict_select(w, tl, budget, sink=2, recent=8)
    moved = (keep != torch.arange(budget, device=gpu)) & (keep >= 0)
    assert int(moved[0, 0, :256].sum()) > 150 and int(moved[1, 0].sum()) < 30 and not bool(moved[2].any())
    want = [_expected(_raw(c), keep, tables, hw) for c in (k, v)]
    evict_move(keep, tl, tables, k, v)
    assert torch.equal(_raw(k), want[0]) and torch.equal(_raw(v), want[1])


def test_move_of_positions(gpu):
    """Stored positions move, appended slots get theirs, nothing past the new end is written."""
    lens, kept, seen, budget = [80, 64, 30], [64, 64, 20], [500, 64, 45], 64
    k, v = _caches(gpu, 20, 16, 2, 64, torch.bfloat16, "paired")
    tables = torch.arange(18, dtype=torch.int32, device=gpu).view(3, 6)
    g = torch.Generator(device=gpu).manual_seed(2)
    pos = torch.stack([torch.randperm(96, generator=g, device=gpu) for _ in range(6)]).view(3, 2, 96).to(torch.int32)
    w = _weights(gpu, 3, 2, 96, 22, "plain")
    i32 = [torch.tensor(x, dtype=torch.int32, device=gpu) for x in (lens, kept, seen)]
    keep, new = evict_select(w, i32[0], budget, sink=4, recent=8, positions=pos, kept=i32[1], seen=i32[2])
    want = pos.cpu().numpy().copy()
    for b in range(3):
        n = min(lens[b], budget)
        for h in range(2):
            at = oracle.slot_positions(lens[b], pos[b, h].cpu().numpy(), kept[b], seen[b])
            want[b, h, :n] = at[keep[b, h, :n].cpu().numpy()]
    evict_move(keep, i32[0], tables, k, v, weights=w, positions=pos, kept=i32[1], seen=i32[2])
    assert np.array_equal(pos.cpu().numpy(), want)
    assert new.tolist() == [64, 64, 30]


def test_nothing_to_do(gpu):
    k, v = _caches(gpu, 4, 16, 2, 64, torch.float16, "native")
    before = k.clone(), v.clone()
    empty = torch.zeros(0, 2, 64, device=gpu)
    lens = torch.zeros(0, dtype=torch.int32, device=gpu)
    keep, new = evict_select(empty, lens, 8)
    assert keep.shape == (0, 2, 8) and new.shape == (0,)
    evict_move(keep, lens, torch.zeros(0, 4, dtype=torch.int32, device=gpu), k, v)
    assert torch.equal(_raw(k), _raw(before[0])) and torch.equal(_raw(v), _raw(before[1]))


def test_keys_that_differ_below_their_sign_up_to_nan(gpu):
    """The search's candidates past the greatest key: no negative weight, and NaN as the threshold."""
    w = _weights(gpu, 1, 3, 3000, 31, "plain")
    w[0, 0, ::3] = float("nan")
    w[0, 1, ::3] = float("inf")
    w[0, 2, ::2] = 0.0
    _check_select(w, [3000], 700, 4, 64)
    _check_select(w, [3000], 1200, 4, 64)


@pytest.mark.parametrize("budget", [300, 1500, 2500, 3900])
def test_weights_a_few_last_bits_apart(gpu, budget):
    """More keys of one bin than are searched apart, next to keys a few units above them."""
    g = torch.Generator(device=gpu).manual_seed(6)
    steps = torch.tensor([0, 1, 2, 3, 8, 9, 11, 5000], device=gpu)
    w = 1.0 + steps[torch.randint(0, 8, (1, 2, 4000), generator=g, device=gpu)] * 2.0**-23
    w[0, 1, ::2] = 5.0
    _check_select(w.float(), [4000], budget, 2, 30)


def _select_ms(w, lens, budget):
    """Median time of the kernel."""
    tl = torch.tensor(lens, dtype=torch.int32, device=w.device)
    for _ in range(5):
        evict_select(w, tl, budget, sink=4, recent=256)
    torch.cuda.synchronize()
    ops.KernelTimer.reset()
    with ops.KernelTimer() as timer:
        for _ in range(31):
            evict_select(w, tl, budget, sink=4, recent=256)
        torch.cuda.synchronize()
    return sorted(timer.durations("cf_evict_select"))[15]


@pytest.mark.parametrize("s, b, budget", [(30000, 4, 4096), (16000, 4, 4096)])
def test_slots_past_the_sequence_do_not_slow_the_search(gpu, s, b, budget):
    """The histogram's bins come from the keys of the sequence: a sequence that
    ends before its buffer, whose last waves hold nothing, is searched as one that
    fills it.  Weights of one binade: with a range that took in the empty slots
    their leading bits, all alike, chose one bin for all of them, and a shorter
    sequence took half as long again."""
    w = 1.0 + torch.rand(b, 8, s, generator=torch.Generator(device=gpu).manual_seed(8), device=gpu)
    _check_select(w[:1, :2], [s * 9 // 10], budget, 4, 256)
    whole = _select_ms(w, [s] * b, budget)
    for n in (s * 9 // 10, s * 7 // 10, s // 2):
        assert _select_ms(w, [n] * b, budget) <= 1.3 * whole, n
