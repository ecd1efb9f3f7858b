"""Edges of caches with a scale for each block and head: scales that are not finite, and blocks whose scales lie far
apart, in the attention calls."""

from __future__ import annotations

import math

import pytest
import torch

from block_scaled_util import filled
from cf_hip.layout import alloc_kv_cache, alloc_kv_scales
from kernels.block_scaled_kv import write_kv_blocks
from kernels.paged_attention import paged_attention_tensors

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
