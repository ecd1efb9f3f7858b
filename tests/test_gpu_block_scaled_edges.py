"""Edges of caches with a scale for each block and head: scales that are not finite, and blocks whose scales lie far
apart, in the attention calls."""

from __future__ import annotations

import math

import pytest
import torch

from block_scaled_util import assert_attended, attend_ref, dense, filled
from cf_hip import ops
from cf_hip.layout import alloc_kv_cache, alloc_kv_scales
from kernels.block_scaled_kv import write_kv_blocks
from kernels.paged_attention import chunked_prefill_attention, paged_attention_tensors

pytestmark = pytest.mark.gpu

E4M3, I8 = torch.float8_e4m3fn, torch.int8
KV = [E4M3, I8]
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _device_cache(k, v, ks, vs, layout):
    nb, bs, h, d = k.shape
    caches = alloc_kv_cache(nb, bs, h, d, k.dtype, "cuda", layout)
    for c, x in zip(caches, (k, v)):
        c.view(torch.uint8).copy_(x.view(torch.uint8).cuda())
    scales = alloc_kv_scales(nb, h, "cuda")
    for s, x in zip(scales, (ks, vs)):
        s.copy_(x)
    return *caches, *scales


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("qt", [BF16, F16, F32])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("layout, hq, dim, bs", [("paired", 8, 128, 16), ("token_major", 8, 64, 16), ("native", 12, 64, 16),
                                                 ("paired", 8, 40, 16), ("token_major", 4, 64, 8)])
def test_decode_not_finite(dtype, qt, side, layout, hq, dim, bs):
    """A visible block of a NaN scale makes NaN of its head's group in the sequences that see it, wherever it lies and
    also where a wave or the whole sequence sees no other; the rest is that of the call without it, bit for bit."""
    gen = torch.Generator().manual_seed(dim + hq)
    lens = [7, bs, 40, 40, 3001, 3001, 2000, 500, bs]
    blocks = [-(-n // bs) for n in lens]
    at = [sum(blocks[:i]) for i in range(len(lens) + 1)]
    tables = [list(range(at[i], at[i + 1])) + [-1] * (max(blocks) - blocks[i]) for i in range(len(lens))]
    k, ks = filled(at[-1], bs, 2, dim, dtype, gen)
    v, vs = filled(at[-1], bs, 2, dim, dtype, gen)
    q = torch.randn(len(lens), hq, dim, generator=gen).to(qt).cuda()
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, layout)

    def run():
        return paged_attention_tensors(q, kc, vc, _i32(tables), _i32(lens), bs, k_scale=ksd, v_scale=vsd)

    clean = run()
    assert bool(clean.isfinite().all())
    scales = ksd if side == "k" else vsd
    seen = {0: [0], 2: [0], 3: [blocks[3] - 1], 4: range(60), 5: [77], 6: range(blocks[6]), 8: [0]}
    for i, js in seen.items():
        scales[[tables[i][j] for j in js], 1] = math.nan
    nan = torch.zeros(len(lens), hq, dtype=torch.bool)
    nan[list(seen), hq // 2:] = True
    got = run()
    assert torch.equal(got.isnan().any(-1).cpu(), nan) and torch.equal(got.isnan().all(-1).cpu(), nan)
    assert torch.equal(got[~nan.cuda()], clean[~nan.cuda()])


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("qt", [BF16, F32])
def test_decode_not_finite_shared_prefix(dtype, qt):
    """The same in blocks that several sequences share, and in a member's own ones."""
    gen = torch.Generator().manual_seed(6)
    prefix = list(range(8))
    tables = [prefix + [8 + 3 * b, 9 + 3 * b, 10 + 3 * b] for b in range(5)]
    lens = [160, 128, 176, 150, 133]
    k, ks = filled(24, 16, 2, 128, dtype, gen)
    v, vs = filled(24, 16, 2, 128, dtype, gen)
    q = torch.randn(5, 8, 128, generator=gen).to(qt).cuda()
    for bad, members in (([0, 1, 2], [0, 1, 2, 3, 4]), ([14, 15, 16], [2]), (prefix, [0, 1, 2, 3, 4])):
        kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, "paired")
        args = (q, kc, vc, _i32(tables), _i32(lens))
        kw = dict(k_scale=ksd, v_scale=vsd, shared_prefix_lens=_i32([0, 128, 128, 128, 128]))
        clean = paged_attention_tensors(*args, **kw)
        ksd[bad, 0] = math.nan
        nan = torch.zeros(5, 8, dtype=torch.bool, device="cuda")
        nan[members, :4] = True
        got = paged_attention_tensors(*args, **kw)
        assert torch.equal(got.isnan().any(-1), nan) and torch.equal(got.isnan().all(-1), nan)
        assert torch.equal(got[~nan], clean[~nan])


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("side", ["k", "v"])
def test_decode_written_not_finite(dtype, side):
    """A sequence of one block with a NaN or infinity among its keys or values decodes to NaN."""
    gen = torch.Generator().manual_seed(3)
    kc, vc = alloc_kv_cache(4, 16, 2, 64, dtype, "cuda", "paired")
    ks, vs = alloc_kv_scales(4, 2, "cuda")
    new = [torch.randn(12, 2, 64, generator=gen).bfloat16() for _ in range(2)]
    new[side == "v"][3, 1, 9] = math.inf
    write_kv_blocks(new[0].cuda(), new[1].cuda(), _i32([[2]]), _i32([12]), kc, vc, ks, vs, q_start=_i32([0, 12]))
    q = torch.randn(1, 4, 64, generator=gen).bfloat16().cuda()
    nan = paged_attention_tensors(q, kc, vc, _i32([[2]]), _i32([12]), k_scale=ks, v_scale=vs).isnan()
    assert bool(nan[:, 2:].all()) and not bool(nan[:, :2].any())


def _check_wide(qt, dtype, layout, chunks, hq, hkv, dim, spans, only=None, keys=None, seed=0):
    """Chunks of sequences whose V scales run over 2^first ... 2^last from their first block to their last (spans: a
    pair a sequence).  keys(q, k, tables): changes of the inputs before they go to the GPU."""
    gen = torch.Generator().manual_seed(seed)
    lens = [r + c for r, c in chunks]
    nb = sum(-(-n // 16) for n in lens) + 3
    k, ks = filled(nb, 16, hkv, dim, dtype, gen)
    v, vs = filled(nb, 16, hkv, dim, dtype, gen)
    perm, at, tables = torch.randperm(nb, generator=gen).tolist(), 0, []
    width = max(-(-n // 16) for n in lens)
    for n, (first, last) in zip(lens, spans):
        need = -(-n // 16)
        t = perm[at: at + need]
        at += need
        for j, b in enumerate(t):
            vs[b] *= 2.0 ** round(first + (last - first) * j / max(1, need - 1))
        tables.append(t + [-1] * (width - need))
    start = [sum(r for r, _ in chunks[:n]) for n in range(len(chunks) + 1)]
    q = torch.randn(start[-1], hq, dim, generator=gen).to(qt)
    if keys is not None:
        keys(q, k, tables)
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, layout)
    got = chunked_prefill_attention(q.cuda(), kc, vc, _i32(tables), _i32(lens), _i32(start), 16, dim**-0.5, k_scale=ksd,
                                    v_scale=vsd)
    rows, refs, least = [], [], []
    idx = torch.arange(hq) // (hq // hkv)
    for n, (r, c) in enumerate(chunks):
        if only is not None and n not in only:
            continue
        for i in sorted({0, 1, 15, 16, 31, r // 3, r // 2, r - 17, r - 2, r - 1} & set(range(r))):
            rows.append(start[n] + i)
            refs.append(attend_ref(q[start[n] + i], k, ks, v, vs, tables[n], c + i + 1, dim**-0.5))
            # a weight below fp16's normal numbers: off by 2^-25 of the row's largest weight times scale, by its code
            kd, _ = dense(k, ks, tables[n], c + i + 1, 16)
            blocks = torch.tensor(tables[n])[torch.arange(c + i + 1) // 16]
            p = torch.softmax((q[start[n] + i].double()[:, None] * kd[idx]).sum(-1) * dim**-0.5, -1)
            most = (p * vs.double()[blocks].T[idx]).amax(-1)
            codes = v[blocks, torch.arange(c + i + 1) % 16].float().double().abs().sum(0)[idx]
            least.append(2.0**-25 * most[:, None] * codes)
    # P in fp16 ahead of the product with V, its exponent by a logarithm of up to 2^6 (half of 2^-18), and its subnormals
    refs = [(ref, pv, size, extra) for (ref, pv, size, _), extra in zip(refs, least)]
    assert_attended(got[rows], refs, qt, dim, max(lens), 2.0**-11 + 2.0**-16 + 2.0**-18, f"wide {qt} {dtype} {layout} {chunks}", 1.0)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("layout", ["paired", "native", "token_major"])
@pytest.mark.parametrize("span", [(-20, 20), (20, -20), (-50, 40), (0, 45)])
@pytest.mark.parametrize("hq, hkv, dim", [(8, 2, 128), (4, 4, 64)])
def test_prefill_wide_scales(dtype, layout, span, hq, hkv, dim):
    """V scales that lie far apart along a chunk: a row is as exact as those that it sees make it, whatever later
    blocks hold."""
    _check_wide(BF16, dtype, layout, [(200, 0), (40, 90)], hq, hkv, dim, [span, span], seed=dim)


@pytest.mark.parametrize("dtype", KV)
def test_prefill_wide_scales_fp16(dtype):
    _check_wide(F16, dtype, "paired", [(300, 0), (40, 290)], 8, 2, 128, [(-22, 8), (8, -22)], seed=3)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("span", [(-20, 20), (20, -20)])
def test_prefill_wide_scales_cut_queued_and_long(dtype, span):
    """The same where items are cut and merged, come from the queue, and have more tiles than a workgroup holds the
    scales of."""
    _check_wide(BF16, dtype, "paired", [(20, 3001)], 8, 2, 128, [span], seed=1)
    _check_wide(BF16, dtype, "paired", [(300, 17)] * 6 + [(250, 400)] * 4, 32, 8, 128, [span] * 10, only=(0, 7), seed=2)
    _check_wide(BF16, dtype, "native", [(420, 0)] * 7, 24, 12, 64, [span] * 7, only=(0, 6), seed=4)
    _check_wide(BF16, dtype, "paired", [(160, 12350 + 9 * n) for n in range(7)], 64, 4, 64, [span] * 7, only=(0,), seed=5)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("dim", [64, 128])
def test_prefill_wide_scales_of_no_weight(dtype, dim):
    """Visible blocks of large V scales whose keys the queries turn away from: what is left is exact."""

    def away(q, k, tables):
        # scores of the first three blocks: about -40 in the exponent
        q[:] = (q.float() * 0.2 + 1.0).to(q.dtype)
        for b in tables[0][:3]:
            k[b] = torch.full_like(k[b].float(), -100.0 if dtype == I8 else -256.0).to(dtype)

    _check_wide(BF16, dtype, "paired", [(100, 30)], 8, 2, dim, [(25, -25)], keys=away, seed=6)


@pytest.mark.parametrize("dtype", KV)
def test_prefill_v_scales_of_zero(dtype):
    """Blocks of a V scale of 0 take their weight and add nothing, whatever their codes."""
    gen = torch.Generator().manual_seed(8)
    k, ks = filled(6, 16, 2, 64, dtype, gen)
    v, vs = filled(6, 16, 2, 64, dtype, gen)
    vs[[1, 4]] = 0.0
    vs *= 2.0**-30
    q = torch.randn(90, 4, 64, generator=gen).bfloat16()
    table = [1, 3, 4, 0, 5, 2]
    kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, "paired")
    got = chunked_prefill_attention(q.cuda(), kc, vc, _i32([table]), _i32([90]), _i32([0, 90]), k_scale=ksd, v_scale=vsd)
    refs = [attend_ref(q[i], k, ks, v, vs, table, i + 1, 0.125) for i in range(90)]
    assert not bool(got[:16].any())
    vsd[[1, 4]] = 2.0**-90  # the same below 2^-80
    again = chunked_prefill_attention(q.cuda(), kc, vc, _i32([table]), _i32([90]), _i32([0, 90]), k_scale=ksd, v_scale=vsd)
    assert torch.equal(again, got)
    assert_attended(got, refs, BF16, 64, 90, 2.0**-11 + 2.0**-16 + 2.0**-18, "zero scales", 2.0**-25)


@pytest.mark.parametrize("dtype", KV)
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("scale", [-0.25, -1e-30, -math.inf, math.inf, math.nan])
def test_scales_that_read_as_nan(dtype, side, scale):
    """A negative scale and one that is not finite make NaN of what sees their block and head, in every operator, and
    of nothing else; a scale of -0 is 0."""
    gen = torch.Generator().manual_seed(21)
    for layout, dim in (("paired", 64), ("token_major", 128), ("paired", 40)):
        k, ks = filled(6, 16, 2, dim, dtype, gen)
        v, vs = filled(6, 16, 2, dim, dtype, gen)
        q = torch.randn(40, 8, dim, generator=gen).bfloat16().cuda()
        tables, lens = _i32([[1, 4, 2], [0, 3, 5]]), _i32([40, 33])
        outs = []
        for bad in (None, scale):
            kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, layout)
            if bad is not None:
                (ksd, vsd)[side][4, 1] = bad
            kw = dict(k_scale=ksd, v_scale=vsd)
            out = {"decode": paged_attention_tensors(q[:2], kc, vc, tables, lens, **kw),
                   "gather": ops.paged_gather((kc, vc)[side], tables, 40, scale=(ksd, vsd)[side])}
            if dim != 40:
                out["chunk"] = chunked_prefill_attention(q, kc, vc, tables, lens, _i32([0, 30, 40]), **kw)
            rows = torch.ones(1, 2, dim, dtype=BF16, device="cuda")
            write_kv_blocks(rows, rows, _i32([[1, 4]]), _i32([20]), kc, vc, ksd, vsd)
            out["scales"] = (ksd, vsd)[side].clone()
            outs.append(out)
        nan = {n: torch.zeros(o.shape, dtype=torch.bool, device="cuda") for n, o in outs[0].items()}
        nan["decode"][0, 4:] = True
        nan["gather"][0, 16:32, 1] = True
        nan["scales"][4, 1] = True
        if dim != 40:
            nan["chunk"][6:30, 4:] = True  # positions 16 to 39
        for n, m in nan.items():
            assert torch.equal(outs[1][n].isnan(), m), (n, dim)
            assert torch.equal(outs[1][n][~m], outs[0][n][~m]), (n, dim)
    for s in (0.0, -0.0):
        kc, vc, ksd, vsd = _device_cache(k, v, ks, vs, "paired")
        (ksd, vsd)[side].fill_(s)
        out = paged_attention_tensors(q[:2], kc, vc, tables, lens, k_scale=ksd, v_scale=vsd)
        assert bool(out.isfinite().all()) and (side == 0 or not bool(out.any()))


@pytest.mark.parametrize("layout", ["paired", "token_major"])
@pytest.mark.parametrize("dim", [64, 40])
def test_widened_codes_equal_those_of_one_write(layout, dim):
    """e4m3fn: rows written one at a time under scales that grow have the codes of one write at once, but for codes
    that are subnormal at the end: these are rounded under two scales, and the two roundings (half a step of 2^-9 times
    the scale, and less) leave them a step apart at most."""
    n, gen = 48, torch.Generator().manual_seed(1)
    x = torch.randn(n, 2, dim, generator=gen) * torch.exp2(torch.arange(n).float() / 3)[:, None, None]
    x[5, 0] *= 2.0**-9  # subnormal codes, too
    table, xd, got = _i32([[2, 0, 1]]), x.cuda(), []
    for step in (1, n):
        kc, vc = alloc_kv_cache(3, 16, 2, dim, E4M3, "cuda", layout)
        ks, vs = alloc_kv_scales(3, 2, "cuda")
        for at in range(0, n, step):
            write_kv_blocks(xd[at: at + step], xd[at: at + step], table, _i32([at + step]), kc, vc, ks, vs,
                            q_start=_i32([0, step]))
        got.append((ops.paged_gather(kc, table, n, scale=ks)[0].cpu(), ops.paged_gather(vc, table, n, scale=vs)[0].cpu(),
                    ks.cpu().clone(), vs.cpu().clone()))
    (k1, v1, ks1, vs1), (k2, v2, ks2, vs2) = got
    assert torch.equal(ks1, ks2) and torch.equal(vs1, vs2)
    scale = ks1[[2, 0, 1]].repeat_interleave(16, 0)[..., None]
    normal = x.abs() >= 2.0**-6 * scale
    assert 0 < int((~normal).sum()) < x.numel() // 4
    for a, b in ((k1, k2), (v1, v2)):
        assert torch.equal(a[normal], b[normal])
        assert bool(((a - b).abs() <= 2.0**-9 * scale).all())
