"""Caches in 8 bits with a scale for each block and head: rows written (bit for bit against float32 steps), decode
and chunk attention and gathers over them (against float64, within what their roundings add up to)."""

from __future__ import annotations

import math

import pytest
import torch

from block_scaled_util import (assert_attended, attend_ref, code_bytes, encode, filled, least_scale, write_ref)
from cf_hip import ops
from cf_hip.layout import alloc_kv_cache, alloc_kv_scales, paired_storage
from kernels.block_scaled_kv import write_kv_blocks
from kernels.paged_attention import chunked_prefill_attention, paged_attention, paged_attention_tensors
from python_runtime.engine.block_manager import BlockManager

pytestmark = pytest.mark.gpu

E4M3, I8 = torch.float8_e4m3fn, torch.int8
KV = [E4M3, I8]
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _device_cache(k, v, ks, vs, layout):
    """CPU codes [NB, bs, H, D] and scales in a layout on the GPU; the scales as alloc_kv_scales lays them."""
    nb, bs, h, d = k.shape
    kc, vc = alloc_kv_cache(nb, bs, h, d, k.dtype, "cuda", layout)
    for c, x in ((kc, k), (vc, v)):
        (c.view(torch.uint8) if c.dtype == E4M3 else c).copy_((x.view(torch.uint8) if x.dtype == E4M3 else x).cuda())
    ksd, vsd = alloc_kv_scales(nb, h, "cuda")
    ksd.copy_(ks)
    vsd.copy_(vs)
    return kc, vc, ksd, vsd


def _same_scales(got, want):
    got = got.cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()])


def _same_codes(got, want, scales):
    """Codes bit for bit, and any NaN where the block's scale is NaN (int8 codes there say nothing)."""
    live = ~scales.isnan()[:, None, :, None].expand(want.shape)
    g, w = code_bytes(got.cpu()), code_bytes(want)
    assert torch.equal(g[live], w[live]), int((g[live] != w[live]).sum())


def _check_write(dtype, xt, layout, lens, tables, start, nb=24, bs=16, heads=3, dim=64, seed=0, new=None, spread=1.0,
                 cached=None):
    gen = torch.Generator().manual_seed(seed)
    k, ks = filled(nb, bs, heads, dim, dtype, gen, spread)
    v, vs = filled(nb, bs, heads, dim, dtype, gen, spread)
    if cached is not None:
        cached(k, ks, v, vs)
    total = len(lens) if start is None else start[-1]
    if new is None:
        new = tuple((torch.randn(total, heads, dim, generator=gen) * torch.exp2(spread * torch.randn(total, heads, 1, generator=gen))).to(xt)
                    for _ in range(2))
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, layout)
    k_new, v_new = (x.cuda() for x in new)
    write_kv_blocks(k_new, v_new, _i32(tables).reshape(len(tables), -1), _i32(lens), kc, vc, ksd, vsd,
                    q_start=None if start is None else _i32(start))
    for x, c, s in ((new[0], k, ks), (new[1], v, vs)):
        write_ref(x, tables, lens, start, c, s, bs)
    for got, gs, c, s in ((kc, ksd, k, ks), (vc, vsd, v, vs)):
        _same_scales(gs, s)
        _same_codes(got, c, s)
    return kc, vc, ksd, vsd


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("xt", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["paired", "native", "token_major"])
def test_write_single_rows(dtype, xt, layout):
    """A decode step: rows that start a block, go on in one with and without a wider scale, fill one, sequences
    without tokens, past the table, and with a block outside the cache."""
    tables = [[5, 7], [3, 2], [11, 0], [9, 1], [13, 14], [99, 4], [6, -1], [15, 16]]
    lens = [17, 32, 0, 9, 33, 5, 17, 1]
    _check_write(dtype, xt, layout, lens, tables, None)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("layout", ["paired", "token_major"])
@pytest.mark.parametrize("heads, dim", [(8, 128), (4, 64), (12, 64), (2, 40), (1, 256), (3, 8)])
def test_write_chunks(dtype, layout, heads, dim):
    """Prompts, chunks that go on inside a block, empty ones and single rows in one call."""
    tables = [[0, 1, 2, 3, 4], [5, 6, 7, 8, 9], [10, 11, 12, 13, 14], [15, 16, 17, 18, 19], [20, 21, 22, 23, 23]]
    counts, lens = [50, 0, 33, 1, 16], [50, 12, 40, 30, 64]
    start = [sum(counts[:i]) for i in range(6)]
    _check_write(dtype, BF16, layout, lens, tables, start, heads=heads, dim=dim, seed=heads + dim)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("bs", [1, 5, 8, 32])
def test_write_block_sizes(dtype, bs):
    counts, lens = [13, 1, 7], [13, 20, 23]
    tables = [list(range(i * 8, i * 8 + 8)) for i in range(3)] if bs < 8 else [[0, 1, 2], [3, 4, 5], [6, 7, 8]]
    start = [0, 13, 14, 21]
    _check_write(dtype, F16, "native", lens, tables, start, bs=bs, dim=24, seed=bs)


@pytest.mark.parametrize("dtype", KV)
def test_write_many_sequences(dtype):
    """More than 64 x 64 sequences, most of them without rows."""
    n, gen = 4200, torch.Generator().manual_seed(3)
    counts = [int(c) if c < 3 else 0 for c in torch.randint(0, 40, (n,), generator=gen)]
    start = [0]
    for c in counts:
        start.append(start[-1] + c)
    with_rows = [i for i in range(n) if counts[i]]
    tables = [[0]] * n
    for j, i in enumerate(with_rows):
        tables[i] = [j]
    lens = [counts[i] + (i % 5) for i in range(n)]
    _check_write(dtype, BF16, "paired", lens, tables, start, nb=len(with_rows), heads=1, dim=64)


@pytest.mark.parametrize("dtype", KV)
def test_write_rows_out_of_reach(dtype):
    """More rows than tokens (the first ones have no position), rows past the table, and starts that do not begin
    at row 0."""
    tables = [[1, 2], [3, 4]]
    _check_write(dtype, F32, "paired", [5, 40], tables, [0, 9, 45])
    _check_write(dtype, F32, "paired", [20, 3], tables, [4, 24, 27], new=tuple(torch.randn(40, 3, 64) for _ in range(2)))


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("size", [0.0, 1e-30, 2.0**-45, 1e-10, 1e10, 3e38])
def test_write_magnitudes(dtype, size):
    """Zeros, values below the least scale, and the largest: no code overflows."""
    new = tuple(torch.randn(20, 3, 64).clamp(-1, 1) * size for _ in range(2))
    kc, _, ksd, _ = _check_write(dtype, F32, "paired", [20], [[3, 8]], [0, 20], new=new)
    assert not bool(kc.float().isnan().any()) and bool((ksd > 0).all())


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_write_not_finite(dtype, bad):
    """The block and head of a NaN or infinity reads as NaN, later rows included, until it starts anew."""
    x = torch.randn(20, 3, 64)
    x[4, 1, 7] = bad
    kc, vc, ks, vs = _check_write(dtype, BF16, "paired", [20], [[3, 8]], [0, 20], new=(x.bfloat16(), torch.randn(20, 3, 64).bfloat16()))
    assert ks.isnan().nonzero().tolist() == [[3, 1]]
    out = ops.paged_gather(kc, _i32([[3, 8]]), 20, scale=ks)
    assert bool(out[0, :16, 1].isnan().all()) and not bool(out[0, :, 0].isnan().any()) and not bool(out[0, 16:].isnan().any())
    row = torch.ones(1, 3, 64, dtype=BF16, device="cuda")
    write_kv_blocks(row, row, _i32([[3, 8]]), _i32([6]), kc, vc, ks, vs)
    assert bool(ks[3, 1].isnan())
    write_kv_blocks(row, row, _i32([[3, 8]]), _i32([1]), kc, vc, ks, vs)
    assert float(ks[3, 1]) == least_scale(1.0, dtype)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("layout", ["paired", "token_major"])
@pytest.mark.parametrize("dim", [64, 128])
def test_write_behind_any_scale(dtype, layout, dim):
    """Rows behind cached ones of scales that no write chose: not powers of two, wider than the rows need, past
    2^126, and codes of every value."""

    def cached(k, ks, v, vs):
        every = torch.arange(256, dtype=torch.uint8).repeat(k[0].numel() // 256)
        for c, s in ((k, ks), (v, vs)):
            code_view = c.view(torch.uint8) if dtype == E4M3 else c
            code_view[2] = every.view(code_view.dtype).reshape(c[2].shape)
            s[:, 0] *= 1.37
            s[:, 1] *= 61.0
            s[1] = torch.tensor([2.0**126, 1.3 * 2.0**126, 2.0**127, 2.0**125])
            s[2] = torch.tensor([0.7e-3, 1e-3, 2.0**-9, 3.0])

    start = [0, 3, 13, 14, 30]
    _check_write(dtype, BF16, layout, [10, 17, 12, 30], [[0, 4], [1, 5], [2, 6], [3, 7]], start, heads=4, dim=dim, cached=cached)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("xt", [BF16, F32])
def test_write_rows_off_their_alignment(dtype, xt):
    """New rows that begin one element behind a 16-byte boundary, and keys and values of different layouts."""
    gen = torch.Generator().manual_seed(11)
    flat = torch.randn(2, 40 * 2 * 64 + 1, generator=gen).to(xt)
    k, ks = filled(6, 16, 2, 64, dtype, gen)
    v, vs = filled(6, 16, 2, 64, dtype, gen)
    tables, lens, start = [[0, 1], [2, 3], [5, 4]], [20, 20, 13], [0, 20, 27, 40]
    for first in (0, 1):
        new = [f.cuda()[first : first + 40 * 2 * 64].view(40, 2, 64) for f in flat]
        kc, _, ksd, _ = _device_cache(k, v, ks, vs, "token_major")
        _, vc, _, vsd = _device_cache(k, v, ks, vs, "native")
        write_kv_blocks(new[0], new[1], _i32(tables), _i32(lens), kc, vc, ksd, vsd, q_start=_i32(start))
        for x, got, gs, c, s in ((new[0], kc, ksd, k.clone(), ks.clone()), (new[1], vc, vsd, v.clone(), vs.clone())):
            write_ref(x.cpu(), tables, lens, start, c, s, 16)
            _same_scales(gs, s)
            _same_codes(got, c, s)


@pytest.mark.parametrize("dtype", KV)
def test_write_row_by_row(dtype):
    """A block filled one row at a time, each wider than the last: values stay within what the widenings add up to
    (e4m3: exact but for subnormals; int8: half a step of every scale since), and e4m3 equals one write at once."""
    heads, dim, n = 2, 64, 32
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(n, heads, dim, generator=gen) * torch.exp2(torch.arange(n).float() / 3)[:, None, None]
    k, v = alloc_kv_cache(3, 16, heads, dim, dtype, "cuda", "paired")
    ks, vs = alloc_kv_scales(3, heads, "cuda")
    xd = x.cuda()
    for i in range(n):
        write_kv_blocks(xd[i: i + 1], xd[i: i + 1], _i32([[2, 1]]), _i32([i + 1]), k, v, ks, vs)
    got = ops.paged_gather(k, _i32([[2, 1]]), n, scale=ks)[0].cpu()
    assert torch.equal(got, ops.paged_gather(v, _i32([[2, 1]]), n, scale=vs)[0].cpu())
    for blk, at in ((2, slice(0, 16)), (1, slice(16, 32))):
        s = ks[blk].cpu()[None, :, None]
        rows = x[at]
        if dtype == E4M3:
            tol = 2.0**-4 * rows.abs() + 2.0**-10 * s * 2
        else:  # scales grow by 2^(1/3) a row: half steps 1/2 (1 + 2^-1/3 + 2^-2/3 + ...) < 2.5 of the last
            tol = 2.5 * s
        assert bool(((got[at] - rows).abs() <= tol).all())
    whole = alloc_kv_cache(3, 16, heads, dim, dtype, "cuda", "paired")
    ws = alloc_kv_scales(3, heads, "cuda")
    write_kv_blocks(xd, xd, _i32([[2, 1]]), _i32([n]), *whole, *ws, q_start=_i32([0, n]))
    assert torch.equal(ws[0][1:], ks[1:])


def test_write_strided_inputs():
    """Rows, tables, lengths, caches and scales that are views of wider tensors."""
    gen = torch.Generator().manual_seed(7)
    heads, dim = 4, 64
    qkv = torch.randn(6, 3 * heads, 2 * dim, generator=gen).bfloat16().cuda()
    k_new, v_new = qkv[:, heads: 2 * heads, ::2], qkv[:, 2 * heads:, 1::2]
    wide = _i32([[0, 9, 1, 9], [2, 9, 3, 9], [4, 9, 5, 9]])
    lens = _i32([[20, 0], [17, 0], [4, 0]])[:, 0]
    slab = torch.zeros(12, 2, 2, heads, 16, dim, dtype=I8, device="cuda")
    kc, vc = slab[:, 1, 0].permute(0, 2, 1, 3), slab[:, 1, 1].permute(0, 2, 1, 3)
    scales = torch.zeros(12, heads, 3, device="cuda")
    start = _i32([0, 5, 2, 5, 3, 5, 6, 5])[::2]  # 0, 2, 3, 6
    write_kv_blocks(k_new, v_new, wide[:, ::2], lens, kc, vc, scales[:, :, 0], scales[:, :, 2], q_start=start)
    for c, s, x in ((kc, scales[:, :, 0], k_new), (vc, scales[:, :, 2], v_new)):
        codes, sc = torch.zeros(12, 16, heads, dim, dtype=I8), torch.zeros(12, heads)
        write_ref(x.cpu(), [[0, 1], [2, 3], [4, 5]], [20, 17, 4], [0, 2, 3, 6], codes, sc, 16)
        _same_scales(s, sc)
        _same_codes(c, codes, sc)
    assert not bool(slab[:, 0].any()) and not bool(scales[:, :, 1].any())


# ---- attention ---------------------------------------------------------------------------


def _scattered(lens, nb, gen, width=None, bs=16):
    perm = torch.randperm(nb, generator=gen).tolist()
    rows, at = [], 0
    for n in lens:
        need = -(-n // bs)
        rows.append(perm[at: at + need])
        at += need
    assert at <= nb
    width = width or max([1] + [len(r) for r in rows])
    return [r + [-1] * (width - len(r)) for r in rows]


def _check_decode(qt, dtype, layout, lens, hq, hkv, dim, seed=0, bs=16, tables=None, nb=None, spread=2.0, call=None, scale=None,
                  shared=None):
    gen = torch.Generator().manual_seed(seed)
    nb = nb or sum(-(-n // bs) for n in lens) + 3
    k, ks = filled(nb, bs, hkv, dim, dtype, gen, spread)
    v, vs = filled(nb, bs, hkv, dim, dtype, gen, spread)
    q = torch.randn(len(lens), hq, dim, generator=gen).to(qt)
    tables = tables or _scattered(lens, nb, gen, bs=bs)
    scale = 1 / math.sqrt(dim) / 2 if scale is None else scale
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, layout)
    got = (call or paged_attention_tensors)(q.cuda(), kc, vc, _i32(tables), _i32(lens), bs, scale, k_scale=ksd, v_scale=vsd,
                                            shared_prefix_lens=shared, partition_tokens=512 // bs * bs)
    refs = [attend_ref(q[b], k, ks, v, vs, tables[b], lens[b], scale, bs) for b in range(len(lens))]
    # two bf16 terms of P (float32 queries: three)
    assert_attended(got, refs, qt, dim, max(lens), 2.0**-23 if qt == F32 else 2.0**-16, f"{qt} {dtype} {layout} {hq}/{hkv} x {dim}")
    return got


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("qt", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["paired", "native", "token_major"])
@pytest.mark.parametrize("hq, hkv, dim", [(8, 2, 128), (12, 12, 64)])
def test_decode(dtype, qt, layout, hq, hkv, dim):
    _check_decode(qt, dtype, layout, [1, 16, 17, 0, 33, 100, 250, 31], hq, hkv, dim, seed=dim)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("hq, hkv, dim, bs, layout", [
    (6, 2, 128, 16, "paired"), (4, 4, 32, 16, "native"), (8, 2, 96, 16, "token_major"), (8, 2, 64, 8, "paired"),
    (4, 1, 40, 5, "native"), (32, 1, 64, 16, "paired"), (16, 1, 128, 16, "paired"), (2, 1, 64, 16, "paired")])
def test_decode_shapes(dtype, hq, hkv, dim, bs, layout):
    """Groups, head dims and block sizes of both kernels."""
    for qt in (BF16, F32):
        _check_decode(qt, dtype, layout, [3, 0, 70, 301], hq, hkv, dim, seed=hq, bs=bs)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("qt", [BF16, F32])
def test_decode_long(dtype, qt):
    """A sequence split over many waves, beside short ones."""
    _check_decode(qt, dtype, "paired", [6001, 5, 640], 8, 2, 64, seed=5, spread=3.0)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("hq, dim", [(4, 64), (6, 64)])
def test_decode_bad_blocks(dtype, hq, dim):
    """Ids outside the cache draw nothing, whatever the scales of the block that stands in for them; lengths past
    the table are cut; a row whose every block is bad is zero."""
    gen = torch.Generator().manual_seed(2)
    hkv = 2
    k, ks = filled(8, 16, hkv, dim, dtype, gen)
    v, vs = filled(8, 16, hkv, dim, dtype, gen)
    ks[0], vs[0] = math.nan, math.inf  # block 0 stands in for bad ones
    tables = [[1, -1, 2], [9, 3, -5], [-1, 100, 8], [4, 5, 6], [7, -1, -1]]
    lens = [48, 40, 48, 1000, 16]
    q = torch.randn(5, hq, dim, generator=gen).bfloat16()
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, "paired")
    got = paged_attention_tensors(q.cuda(), kc, vc, _i32(tables), _i32(lens), k_scale=ksd, v_scale=vsd)
    refs = [attend_ref(q[b], k, ks, v, vs, tables[b], lens[b], dim**-0.5) for b in range(5)]
    assert_attended(got, refs, BF16, dim, 48, 2.0**-16, "bad blocks")
    assert not bool(got[2].any())


@pytest.mark.parametrize("dtype", KV)
def test_decode_masked_slots_may_hold_anything(dtype):
    """Codes past a sequence's end (NaN codes among them) and scales of blocks past it have no say."""
    gen = torch.Generator().manual_seed(4)
    k, ks = filled(6, 16, 2, 128, dtype, gen)
    v, vs = filled(6, 16, 2, 128, dtype, gen)
    lens, tables = [20, 37], [[1, 2, 3], [4, 5, 0]]
    q = torch.randn(2, 8, 128, generator=gen).bfloat16()
    refs = [attend_ref(q[b], k, ks, v, vs, tables[b], lens[b], 128**-0.5) for b in range(2)]
    for c in (k, v):
        raw = c.view(torch.uint8)
        raw[2, 4:] = 0x7F
        raw[0, 5:] = 0x7F
    ks[3], vs[3] = math.nan, math.nan
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, "paired")
    got = paged_attention_tensors(q.cuda(), kc, vc, _i32(tables), _i32(lens), k_scale=ksd, v_scale=vsd)
    assert_attended(got, refs, BF16, 128, 37, 2.0**-16, "masked slots")


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("qt", [BF16, F32])
def test_decode_shared_prefix(dtype, qt):
    """The shared-prefix statement changes how blocks are read, not the result."""
    gen = torch.Generator().manual_seed(6)
    prefix = list(range(8))
    tables = [prefix + [8 + 3 * b, 9 + 3 * b, 10 + 3 * b] for b in range(5)]
    lens = [160, 128, 176, 150, 133]
    shared = _i32([0, 128, 128, 128, 128])
    _check_decode(qt, dtype, "paired", lens, 8, 2, 128, seed=8, tables=tables, nb=24, shared=shared)


def test_decode_wide_scales():
    """Blocks whose scales lie 2^40 apart, and V scales beyond what 16-bit floats hold."""
    gen = torch.Generator().manual_seed(9)
    for dtype in KV:
        k, ks = filled(8, 16, 2, 128, dtype, gen)
        v, vs = filled(8, 16, 2, 128, dtype, gen)
        vs *= torch.exp2(torch.linspace(-60, 60, 8))[:, None]
        q = torch.randn(3, 8, 128, generator=gen).bfloat16()
        tables, lens = [[0, 1, 2], [3, 4, 5], [7, 6, 0]], [48, 40, 48]
        kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, "paired")
        got = paged_attention_tensors(q.cuda(), kc, vc, _i32(tables), _i32(lens), k_scale=ksd, v_scale=vsd)
        refs = [attend_ref(q[b], k, ks, v, vs, tables[b], lens[b], 128**-0.5) for b in range(3)]
        assert_attended(got, refs, BF16, 128, 48, 2.0**-16, "wide scales")


def test_decode_strided_scales():
    """Scales of one layer of a slab's [NB, L, H], and broadcast ones."""
    gen = torch.Generator().manual_seed(10)
    k, ks = filled(6, 16, 2, 64, I8, gen)
    v, _ = filled(6, 16, 2, 64, I8, gen)
    q = torch.randn(2, 4, 64, generator=gen).half()
    tables, lens = [[0, 1, 2], [3, 4, 5]], [40, 48]
    kc, vc, _, _ = _device_cache(k, v, ks, ks, "paired")
    slab = torch.full((6, 3, 2), math.nan, device="cuda")
    slab[:, 1] = ks.cuda()
    one = torch.full((1, 1), 0.02, device="cuda").expand(6, 2)
    got = paged_attention_tensors(q.cuda(), kc, vc, _i32(tables), _i32(lens), k_scale=slab[:, 1], v_scale=one)
    refs = [attend_ref(q[b], k, ks, v, torch.full((6, 2), 0.02), tables[b], lens[b], 0.125) for b in range(2)]
    assert_attended(got, refs, F16, 64, 48, 2.0**-16, "strided scales")


def test_decode_dict_api_plan_and_noalloc():
    """The other decode entry points take block scales, too, with the same result."""
    gen = torch.Generator().manual_seed(11)
    k, ks = filled(6, 16, 2, 128, I8, gen)
    v, vs = filled(6, 16, 2, 128, I8, gen)
    q = torch.randn(2, 8, 128, generator=gen).bfloat16().cuda()
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, "paired")
    tables, lens = [[0, 1, 2], [3, 4, 5]], [40, 48]
    want = paged_attention_tensors(q, kc, vc, _i32(tables), _i32(lens), k_scale=ksd, v_scale=vsd)
    out = paged_attention(q, kc, vc, {"a": tables[0], "b": tables[1]}, {"a": 40, "b": 48}, k_scale=ksd, v_scale=vsd)
    assert torch.equal(torch.stack([out["a"], out["b"]]), want)
    args = (q, kc, vc, _i32(tables), _i32(lens), 128**-0.5, 16, ksd, vsd)
    assert torch.equal(ops.paged_decode_noalloc(*args), want)
    assert torch.equal(ops.DecodePlan(*args).run(), want)


def _check_prefill(qt, dtype, layout, chunks, hq, hkv, dim, seed=0, spread=1.0, scale=None, bad=None, only=None):
    """chunks: (rows, cached tokens); only: the chunks whose outermost rows are compared (all rows' samples of all)."""
    gen = torch.Generator().manual_seed(seed)
    lens = [r + c for r, c in chunks]
    nb = sum(-(-n // 16) for n in lens) + 3
    k, ks = filled(nb, 16, hkv, dim, dtype, gen, spread)
    v, vs = filled(nb, 16, hkv, dim, dtype, gen, spread)
    tables = _scattered(lens, nb, gen)
    if bad is not None:
        bad(tables, ks, vs)
    start = [0]
    for r, _ in chunks:
        start.append(start[-1] + r)
    q = torch.randn(start[-1], hq, dim, generator=gen).to(qt)
    scale = dim**-0.5 if scale is None else scale
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, layout)
    got = chunked_prefill_attention(q.cuda(), kc, vc, _i32(tables), _i32(lens), _i32(start), 16, scale, k_scale=ksd, v_scale=vsd)
    rows, refs = [], []
    for n, (r, c) in enumerate(chunks):
        if only is not None and n not in only:
            continue
        sample = {0, r - 1} if only is not None else {0, 1, r // 2, r - 2, r - 1}
        for i in sorted(sample & set(range(r))) if r > 12 else range(r):
            rows.append(start[n] + i)
            refs.append(attend_ref(q[start[n] + i], k, ks, v, vs, tables[n], c + i + 1, scale))
    # P in fp16 ahead of the product with V, and its subnormals
    assert_attended(got[rows], refs, qt, dim, max(lens), 2.0**-11 + 2.0**-16, f"prefill {qt} {dtype} {layout} {chunks}", 2.0**-25)
    return got


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("qt", [BF16, F16])
@pytest.mark.parametrize("layout", ["paired", "native", "token_major"])
@pytest.mark.parametrize("hq, hkv, dim", [(8, 2, 128), (12, 12, 64), (4, 4, 128), (16, 1, 64)])
def test_prefill(dtype, qt, layout, hq, hkv, dim):
    _check_prefill(qt, dtype, layout, [(1, 0), (5, 30), (40, 0), (17, 100), (33, 15)], hq, hkv, dim, seed=dim + hq)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("qt", [BF16, F16])
def test_prefill_cut_items(dtype, qt):
    """A short chunk behind a long prefix: pieces and their merge."""
    _check_prefill(qt, dtype, "paired", [(20, 3001)], 8, 2, 128, seed=1, spread=2.0)
    _check_prefill(qt, dtype, "token_major", [(7, 1500), (3, 90)], 8, 2, 64, seed=2)


@pytest.mark.parametrize("dtype", KV)
def test_prefill_queued(dtype):
    """More items than resident workgroups: the plan and its queue."""
    _check_prefill(BF16, dtype, "paired", [(300, 17)] * 6 + [(250, 400)] * 4, 32, 8, 128, seed=3)
    _check_prefill(F16, dtype, "native", [(420, 0)] * 7, 24, 12, 64, seed=4)


@pytest.mark.parametrize("dtype", KV)
def test_prefill_long_items(dtype):
    # more tiles in one item than a workgroup holds the scales of (256), with V scales that rise along one sequence
    # and fall along another, and some that are invalid far along
    def slopes(tables, ks, vs):
        blocks = len(tables[0])
        for j in range(blocks):
            vs[tables[0][j]] *= 2.0 ** (j * 12 // blocks)
            vs[tables[6][j]] *= 2.0 ** (12 - j * 12 // blocks)
        for j in (300, 513, 700):
            tables[6][j] = -1

    _check_prefill(F16, dtype, "paired", [(160, 12350 + 9 * n) for n in range(7)], 64, 4, 64, seed=9, bad=slopes, only=(0, 6))


@pytest.mark.parametrize("dtype", KV)
def test_prefill_bad_blocks(dtype):
    """Ids outside the cache are not seen, whatever the scales of the block that stands in for them."""
    def bad(tables, ks, vs):
        tables[0][1] = -1
        tables[1][0], tables[1][2] = 10_000, -7
        used = {b for t in tables for b in t}
        for t in tables:  # block 0 stands in for them; keep it for that
            for j, b in enumerate(t):
                if b == 0:
                    t[j] = next(i for i in range(len(ks)) if i not in used)
                    used.add(t[j])
        ks[0], vs[0] = math.nan, math.inf

    _check_prefill(BF16, dtype, "paired", [(9, 40), (12, 60), (10, 5)], 8, 2, 128, seed=5, bad=bad)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("scale", [0.0, -0.05, 1e-20, 3.0])
def test_prefill_scales_of_scores(dtype, scale):
    _check_prefill(F16, dtype, "paired", [(9, 40), (30, 0)], 8, 2, 128, seed=6, scale=scale, spread=0.3)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("order", [1, -1])
def test_prefill_varied_v_scales(dtype, order):
    """V scales that grow or fall by 2^16 along the sequence, and ones beyond 16-bit floats."""
    def bad(tables, ks, vs):
        for t in tables:
            for j, b in enumerate(t):
                vs[b] *= 2.0 ** (order * 16 * j / len(t))

    _check_prefill(BF16, dtype, "paired", [(33, 200), (70, 0)], 8, 2, 128, seed=7, bad=bad)

    def far(tables, ks, vs):
        for n, t in enumerate(tables):
            for b in t:
                vs[b] *= 2.0 ** (60 * order * (2 * n - 1))

    _check_prefill(BF16, dtype, "paired", [(33, 20), (20, 30)], 8, 2, 64, seed=8, bad=far)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("layout", ["paired", "token_major"])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("at, cached", [(20, 0), (5, 40), (33, 21)])
def test_prefill_not_finite(dtype, layout, side, at, cached):
    """A NaN among a chunk's rows: NaN from the first row that sees its block on, in its head's group alone, and the
    rows before it as if it were not there."""
    gen = torch.Generator().manual_seed(14)
    rows, heads, dim = 50, 2, 128
    n = rows + cached
    tables = [torch.randperm(10, generator=gen).tolist()]
    kv = [torch.randn(n, heads, dim, generator=gen).bfloat16() for _ in range(2)]
    k, v = alloc_kv_cache(10, 16, heads, dim, dtype, "cuda", layout)
    ks, vs = alloc_kv_scales(10, heads, "cuda")
    q = torch.randn(rows, 8, dim, generator=gen).bfloat16().cuda()
    outs = []
    for bad in (0.0, math.nan):
        kv[side == "v"][cached + at, 1, 3] = bad
        write_kv_blocks(kv[0].cuda(), kv[1].cuda(), _i32(tables), _i32([n]), k, v, ks, vs, q_start=_i32([0, n]))
        outs.append(chunked_prefill_attention(q, k, v, _i32(tables), _i32([n]), _i32([0, rows]), k_scale=ks, v_scale=vs))
    first = max(0, (cached + at) // 16 * 16 - cached)  # the first row that sees the block
    nan = outs[1].isnan()
    assert bool(nan[first:, 4:].all()) and not bool(nan[:, :4].any()) and not bool(nan[:first].any())
    assert torch.equal(outs[1][:first], outs[0][:first]) and torch.equal(outs[1][:, :4], outs[0][:, :4])


def test_prefill_equals_decode():
    """A chunk of one row is the decode of that row."""
    gen = torch.Generator().manual_seed(12)
    k, ks = filled(8, 16, 2, 128, I8, gen)
    v, vs = filled(8, 16, 2, 128, I8, gen)
    q = torch.randn(2, 8, 128, generator=gen).half().cuda()
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, "paired")
    t, lens = _i32([[0, 1, 2, 3], [4, 5, 6, 7]]), _i32([50, 64])
    a = paged_attention_tensors(q, kc, vc, t, lens, k_scale=ksd, v_scale=vsd)
    b = chunked_prefill_attention(q, kc, vc, t, lens, _i32([0, 1, 2]), k_scale=ksd, v_scale=vsd)
    assert float((a.double() - b.double()).norm() / a.double().norm()) < 2.0**-11 * 2


# ---- gathers ------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("layout", ["paired", "token_major"])
@pytest.mark.parametrize("seq, bs, dim", [(37, 16, 64), (700, 16, 128), (23, 5, 40)])
@pytest.mark.parametrize("out", [None, BF16])
def test_gather(dtype, layout, seq, bs, dim, out):
    gen = torch.Generator().manual_seed(seq)
    mb = -(-seq // bs)
    k, ks = filled(2 * mb + 2, bs, 4, dim, dtype, gen)
    v, vs = filled(2 * mb + 2, bs, 4, dim, dtype, gen)
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, layout)
    tables = torch.randperm(2 * mb + 2, generator=gen)[: 2 * mb].reshape(2, mb).to(torch.int32)
    tables[1, 1] = -1
    for c, s, codes, sc in ((kc, ksd, k, ks), (vc, vsd, v, vs)):
        got = ops.paged_gather(c, tables.cuda(), seq, out_dtype=out, scale=s).cpu()
        t = torch.arange(seq)
        ids = tables[:, t // bs].long()
        want = codes[ids.clamp(min=0), t % bs].float() * sc[ids.clamp(min=0)][..., None]
        want[ids < 0] = 0.0
        assert got.dtype == (out or F32) and torch.equal(got, want.to(got.dtype))


# ---- calls ----------------------------------------------------------------------------------


def _case(seed=0, dtype=I8):
    gen = torch.Generator().manual_seed(seed)
    k, ks = filled(40, 16, 2, 128, dtype, gen)
    v, vs = filled(40, 16, 2, 128, dtype, gen)
    c = dict(zip(("kc", "vc", "ks", "vs"), _device_cache(k, v, ks, vs, "paired")))
    c["rows"] = torch.randn(4, 2, 128, generator=gen).bfloat16().cuda() * 4
    c["q"] = torch.randn(4, 8, 128, generator=gen).bfloat16().cuda()
    c["tables"] = _i32([list(range(10 * i, 10 * i + 10)) for i in range(4)])
    c["lens"] = _i32([150, 9, 33, 160])
    return c


def _step(c):
    write_kv_blocks(c["rows"], c["rows"], c["tables"], c["lens"], c["kc"], c["vc"], c["ks"], c["vs"])
    a = paged_attention_tensors(c["q"], c["kc"], c["vc"], c["tables"], c["lens"], k_scale=c["ks"], v_scale=c["vs"])
    b = chunked_prefill_attention(c["q"], c["kc"], c["vc"], c["tables"], c["lens"], _i32([0, 1, 2, 3, 4]) if "start" not in c
                                  else c["start"], k_scale=c["ks"], v_scale=c["vs"])
    return a, b


def test_another_stream():
    want = _step(_case())
    side = torch.cuda.Stream()
    c = _case()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(c)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_captured_and_replayed():
    """A write and both attentions in a graph, replayed with other rows between eager calls of other sizes; two
    graphs have workspaces of their own."""
    c = _case(1)
    c["start"] = _i32([0, 1, 2, 3, 4])
    kept = {n: c[n].clone() for n in ("kc", "vc", "ks", "vs")} | {n: c[n].clone() for n in ("rows",)}
    _step(c)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(c)
        graphs.append((g, out))
    eager = _case(2)
    for i in range(3):
        for g, out in graphs:
            for n, t in kept.items():
                (c[n].view(torch.uint8) if c[n].dtype == E4M3 else c[n]).copy_(t)
            c["rows"].mul_(1.0 + i)
            g.replay()
            torch.cuda.synchronize()
            got = [o.clone() for o in out]
            codes = c["kc"].clone()
            for n, t in kept.items():
                c[n].copy_(t)
            c["rows"].mul_(1.0 + i)
            want = _step(c)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(codes, c["kc"])
        _step(eager)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("layout, nb", [("paired", 600_000), ("token_major", 1_100_000)])
def test_offsets_past_32_bits(dtype, layout, nb):
    """Blocks at the end of a cache of more than 2^32 bytes hold and give what low ones do, bit for bit."""
    gen = torch.Generator().manual_seed(21)
    lens, start = [50, 33], _i32([0, 37, 70])
    new = [torch.randn(70, 2, 128, generator=gen).to(BF16).cuda() for _ in range(2)]
    q = torch.randn(70, 8, 128, generator=gen).to(BF16).cuda()
    low = [[3, 0, 7, 5], [1, 6, 2, 4]]
    outs = []
    for blocks, first in ((8, 0), (nb, nb - 8)):
        kc, vc = alloc_kv_cache(blocks, 16, 2, 128, dtype, "cuda", layout)
        ks, vs = alloc_kv_scales(blocks, 2, "cuda")
        tables = _i32([[b + first for b in t] for t in low])
        write_kv_blocks(new[0][:26], new[1][:26], tables, _i32([13, 13]), kc, vc, ks, vs, q_start=_i32([0, 13, 26]))
        write_kv_blocks(*new, tables, _i32(lens), kc, vc, ks, vs, q_start=start)
        if blocks == nb:  # and back from there
            mine = [ops.paged_gather(kc, tables, 33, scale=ks)]
            moves = [(nb - 8 + b, b) for b in range(8)] + [(b, nb - 8 + (b + 1) % 8) for b in range(8)]
            for c in ((paired_storage(kc, vc),) if layout == "paired" else (kc, vc)):
                BlockManager.move_blocks(moves, [c])
            BlockManager.move_blocks(moves, [ks, vs])
            tables = _i32(low)
            mine.append(ops.paged_gather(kc, tables, 33, scale=ks))
            assert torch.equal(*mine)
            tables = _i32([[b + first for b in t] for t in low])
            BlockManager.move_blocks([(b, nb - 8 + b) for b in range(8)], [ks, vs])
            for c in ((paired_storage(kc, vc),) if layout == "paired" else (kc, vc)):
                BlockManager.move_blocks([(b, nb - 8 + b) for b in range(8)], [c])
        outs.append([ops.paged_gather(kc, tables, 33, scale=ks), ops.paged_gather(vc, tables, 33, scale=vs),
                     paged_attention_tensors(q[:2], kc, vc, tables, _i32(lens), k_scale=ks, v_scale=vs),
                     paged_attention_tensors(q[:2].float(), kc, vc, tables, _i32(lens), k_scale=ks, v_scale=vs),
                     chunked_prefill_attention(q, kc, vc, tables, _i32(lens), start, k_scale=ks, v_scale=vs)])
        del kc, vc
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert not any(bool(a.isnan().any()) for a in outs[0])


def test_native_path_and_ctypes_agree(monkeypatch):
    """The call path in native code and the one through ctypes."""
    want, c = _step(_case(3)), _case(3)
    table = ops.paged_gather(c["kc"], c["tables"], 40, scale=c["ks"])

    class Slow:
        def __getattr__(self, name):
            return lambda *a: None

    monkeypatch.setattr(ops, "_fast", lambda: Slow())
    assert torch.equal(ops.paged_gather(c["kc"], c["tables"], 40, scale=c["ks"]), table)
    got = _step(c)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_refusals_on_the_device():
    c = _case()
    with pytest.raises(ValueError, match="rank 2"):
        paged_attention_tensors(c["q"], c["kc"], c["vc"], c["tables"], c["lens"], k_scale=c["ks"], v_scale=c["vs"][0])
    with pytest.raises(ValueError, match="expected \\[40, 2\\]"):
        paged_attention_tensors(c["q"], c["kc"], c["vc"], c["tables"], c["lens"], k_scale=c["ks"][:-1], v_scale=c["vs"])
    with pytest.raises(ValueError):
        write_kv_blocks(c["rows"], c["rows"][:3], c["tables"], c["lens"], c["kc"], c["vc"], c["ks"], c["vs"])
    with pytest.raises(ValueError, match="must be on|ROCm"):
        write_kv_blocks(c["rows"], c["rows"], c["tables"].cpu(), c["lens"], c["kc"], c["vc"], c["ks"], c["vs"])
    with pytest.raises(ValueError, match="block scales"):
        ops.paged_gather(c["kc"], c["tables"], 10, scale=c["ks"][0])
    with pytest.raises(NotImplementedError, match="prefill"):
        chunked_prefill_attention(c["q"].float().half()[:, :6], c["kc"], c["vc"], c["tables"], c["lens"], _i32([0, 1, 2, 3, 4]),
                                  k_scale=c["ks"], v_scale=c["vs"])


def test_single_scales_still_work():
    """A scale a head over e4m3 caches is what it was, also as the one row of a one-block cache."""
    gen = torch.Generator().manual_seed(13)
    x = torch.randn(4, 16, 2, 64, generator=gen)
    s = x.abs().amax((0, 1, 3)) / 448
    codes = encode(x, s[:, None], E4M3)
    kc, vc, _, _ = _device_cache(codes, codes, torch.ones(4, 2), torch.ones(4, 2), "paired")
    t = _i32([[0, 1, 2, 3]])
    want = codes.float() * s[:, None]
    assert torch.equal(ops.paged_gather(kc, t, 64, scale=s.cuda())[0].cpu(), want.reshape(64, 2, 64))
    assert torch.equal(ops.paged_gather(kc, t, 64, scale=s.cuda()[None])[0].cpu(), want.reshape(64, 2, 64))
