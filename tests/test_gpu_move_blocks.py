"""Blocks of several tensors copied and rearranged in place: exact moves of bytes."""

from __future__ import annotations

import random
import time

import numpy as np
import pytest
import torch

from cf_hip import ops
from cf_hip.layout import alloc_kv_cache, alloc_kv_scales, paired_storage
from python_runtime.engine.block_manager import BlockManager

pytestmark = pytest.mark.gpu


def _cache(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    raw = torch.randint(0, 256, (*shape[:-1], shape[-1] * torch.empty(0, dtype=dtype).element_size()), generator=g,
                        dtype=torch.uint8)
    return raw.cuda().view(dtype) if dtype != torch.uint8 else raw.cuda()


def _check(caches, moves):
    before = [c.contiguous().view(torch.uint8).clone() for c in caches]
    BlockManager.move_blocks(moves, caches)
    for c, was in zip(caches, before):
        want = was.clone()
        for s, d in np.asarray(moves, dtype=np.int64).reshape(-1, 2).tolist():
            want[d] = was[s]
        assert torch.equal(c.contiguous().view(torch.uint8), want)


SHAPES = [((24, 3, 16, 8), torch.int8), ((24, 2, 5), torch.float32), ((24, 33), torch.uint8), ((24, 4, 64), torch.bfloat16),
          ((24, 1, 1), torch.float32)]


@pytest.mark.parametrize("moves", [
    [(0, 1)], [(3, 3)], [(0, 1), (1, 0)], [(0, 1), (1, 2), (2, 3)], [(2, 3), (1, 2), (0, 1)], [(0, 5), (0, 6), (0, 7), (5, 0)],
    [(i, (i + 1) % 24) for i in range(24)], [(0, i) for i in range(1, 24)], [],
    [(0, 1), (1, 2), (2, 0), (1, 9), (9, 10), (10, 11), (2, 12), (20, 21), (21, 20), (22, 23)],
])
def test_moves(moves):
    _check([_cache(s, t, i) for i, (s, t) in enumerate(SHAPES)], moves)


@pytest.mark.parametrize("seed", range(6))
def test_random_moves(seed):
    """More moves than a launch takes: permutations with long cycles, chains and copies."""
    rng = random.Random(seed)
    nb = rng.choice([64, 900, 2500])
    dst = rng.sample(range(nb), rng.randint(1, nb))
    src = {0: dst[1:] + dst[:1], 1: [rng.randrange(nb) for _ in dst], 2: rng.sample(range(nb), len(dst))}[seed % 3]
    _check([_cache((nb, 48), torch.int8, seed), _cache((nb, 3), torch.float32, seed)], list(zip(src, dst)))


def test_one_long_cycle():
    nb = 1500
    _check([_cache((nb, 80), torch.uint8, 0)], [((i + 1) % nb, i) for i in range(nb)])


def test_many_moves():
    """As many moves as a large pool has, most of them on their own, some in long chains: the host's share of a launch
    does not grow with them."""
    nb, rng = 120_000, random.Random(5)
    ids = rng.sample(range(nb), nb)
    moves = list(zip(ids[:30_000], ids[30_000:60_000]))
    for at in range(60_000, 118_000, 500):
        chain = ids[at : at + 500]
        moves += list(zip(chain[1:], chain[:-1]))
        if at % 1000 == 0:
            moves.append((chain[0], chain[-1]))
    rng.shuffle(moves)
    c = _cache((nb, 16), torch.uint8, 1)
    was = c.clone()
    begin = time.perf_counter()
    BlockManager.move_blocks(np.asarray(moves, dtype=np.int32), [c])
    torch.cuda.synchronize()
    assert time.perf_counter() - begin < 5.0  # (half a millisecond a launch would be 0.1)
    m = torch.tensor(moves).cuda()
    want = was.clone()
    want[m[:, 1]] = was[m[:, 0]]
    assert torch.equal(c, want)


def test_many_tensors_and_large_blocks():
    """More tensors than a launch takes, blocks of more pieces than its grid, and odd sizes and addresses."""
    caches = [_cache((9, 7 + i), torch.uint8, i) for i in range(20)]
    caches.append(_cache((9, 5_000_011), torch.uint8, 30))
    caches.append(_cache((9, 1_000_000), torch.float32, 31))
    caches.append(_cache((10 * 64 + 1,), torch.uint8, 32)[1:].view(10, 64)[:9])
    _check(caches, [(0, 1), (1, 2), (2, 0), (3, 8)])


def test_slab_views():
    """The cache manager's slabs, whose logical order is not that of memory, and blocks with room between them."""
    slab = _cache((12, 2, 3, 8, 16), torch.int8, 1).permute(0, 1, 3, 2, 4)
    apart = _cache((12, 100), torch.uint8, 2)[:, :48]
    _check([slab, apart], [(0, 11), (11, 3), (3, 0), (5, 6)])
    with pytest.raises(ValueError, match="dense"):
        ops.move_blocks([slab[:, :, :4]], [(0, 1)])


def test_slices_of_one_slab():
    """Layers given one by one, scales that lie side by side, and parts of one tensor are apart."""
    slab = _cache((12, 4, 48), torch.uint8, 3)
    ks, vs = alloc_kv_scales(12, 3, "cuda")
    moves = [(0, 11), (11, 3), (3, 0), (5, 6)]
    _check([slab[:, 2], slab[:, 0], slab[:, 3], slab[:, 1]], moves)
    _check([ks, slab[:, 1], vs], moves)
    whole = _cache((30, 64), torch.uint8, 4)
    _check([whole[18:], whole[:12]], moves)
    wide = _cache((24, 4, 48), torch.uint8, 5)
    _check([wide[:12, 0], wide[12:, 0], wide[:, 1]], moves)  # (within one range, in one place of the stride)
    many = _cache((100_000, 64, 8), torch.uint8, 6)
    halves = [part[:, i] for i in range(60) for part in (many[:50_000], many[50_000:])] + [many[:, 60], many[:, 61:]]
    was, begin = many.clone(), time.perf_counter()
    BlockManager.move_blocks([(0, 49_999), (49_999, 7)], halves)
    torch.cuda.synchronize()
    assert time.perf_counter() - begin < 5.0  # (the host's look at 122 tensors does not go block by block)
    for at in (0, 50_000):
        was[at + 7, :60], was[at + 49_999, :60] = was[at + 49_999, :60].clone(), was[at, :60].clone()
    was[7, 60:], was[49_999, 60:] = was[49_999, 60:].clone(), was[0, 60:].clone()
    assert torch.equal(many, was)


def test_paired_cache_with_its_scales():
    k, v = alloc_kv_cache(12, 16, 3, 64, torch.int8, "cuda", "paired")
    for c in (k, v):
        c.copy_(torch.randint(-127, 128, c.shape, dtype=torch.int8))
    ks, vs = alloc_kv_scales(12, 3, "cuda")
    ks.uniform_()
    vs.uniform_()
    was = [t.clone() for t in (k, v, ks, vs)]
    moves = [(0, 5), (5, 11), (11, 0), (3, 4), (3, 9)]
    BlockManager.move_blocks(moves, [paired_storage(k, v), ks, vs])
    for t, w in zip((k, v, ks, vs), was):
        want = w.clone()
        for s, d in moves:
            want[d] = w[s]
        assert torch.equal(t, want)


def test_moves_as_tensor_and_array():
    for moves in (torch.tensor([[0, 1], [1, 0]]), np.array([[0, 1], [1, 0]], dtype=np.int64), ((0, 1), (1, 0))):
        _check([_cache((4, 32), torch.uint8, 1)], moves)
    with pytest.raises(ValueError, match="on the host"):
        ops.move_blocks([_cache((4, 32), torch.uint8, 1)], torch.tensor([[0, 1]]).cuda())
    with pytest.raises(ValueError, match="destination of two"):
        ops.move_blocks([_cache((4, 32), torch.uint8, 1)], [(0, 1), (2, 1)])
    with pytest.raises(ValueError, match="outside"):
        ops.move_blocks([_cache((4, 32), torch.uint8, 1)], [(0, 4)])


def test_equals_copy_blocks():
    """For copy-on-write pairs the two are the same."""
    a, b = _cache((30, 2, 16, 64), torch.float8_e4m3fn, 4), _cache((30, 2, 16, 64), torch.float8_e4m3fn, 4)
    pairs = np.array([[0, 20], [1, 21], [0, 22]], dtype=np.int32)
    BlockManager.copy_blocks(pairs, [a])
    BlockManager.move_blocks(pairs, [b])
    assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_captured():
    """A captured call replays its moves (the ids are part of the launch), also after the list is gone."""
    c = _cache((8, 4096), torch.uint8, 5)
    was = c.clone()
    moves = [(0, 1), (1, 2), (2, 0)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.move_blocks([c], moves)
    del moves
    for i in range(3):
        g.replay()
        torch.cuda.synchronize()
        ops.move_blocks([_cache((8, 64), torch.uint8, 6)], [(3, 4)])
    assert torch.equal(c, was)  # a cycle of three, three times


def test_compaction_keeps_every_request():
    """After compact and move_blocks every table names the bytes it named before."""
    rng = random.Random(3)
    bm = BlockManager(200, 16)
    caches = [_cache((200, 64), torch.int8, 7), _cache((200, 4), torch.float32, 8)]
    for i in range(20):
        bm.allocate(f"r{i}", rng.randint(1, 150))
    for i in range(0, 20, 3):
        bm.free(f"r{i}")
    bm.fork("r1", ["f1", "f2"], 16)
    ids = [f"r{i}" for i in range(20) if i % 3] + ["f1", "f2"]
    held = {r: [c[bm.get_blocks(r)].clone() for c in caches] for r in ids}
    BlockManager.move_blocks(bm.compact(), caches)
    for r in ids:
        for c, was in zip(caches, held[r]):
            assert torch.equal(c[bm.get_blocks(r)].view(torch.uint8), was.view(torch.uint8))
