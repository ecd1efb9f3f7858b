"""Rotary positions and the rotated cache write on the GPU, against float64.

Tolerance of a rotated value before its last rounding, relative to |x1| + |x2|:
the angle is known to half an ulp of its rest in turns (<= 2^-26 turns, 9.4e-8
rad), sine and cosine to 2 ulp (2^-23), scaled and multiplied with one rounding
each and added with another (3 * 2^-24): together 3.9e-7.  Then half a step of
the output's type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cf_hip import layout as L
from kernels.rotary import rotary, rotary_cache_write
from oracle import rotary as oracle

pytestmark = pytest.mark.gpu
TURN = 3.9e-7
HALF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float8_e4m3fn: 2.0**-4}
TINY = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float8_e4m3fn: 2.0**-10}


def _rows(gpu, shape, dtype, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.randn(shape, generator=g, device=gpu).to(dtype)


def _freq(gpu, pairs):
    return (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))).float().to(gpu)


def _f64(t):
    return t.float().cpu().numpy().astype(np.float64)


def _check(got, want, size, dtype, scale=None):
    """`scale`: of the heads, over e4m3fn codes (the division rounds once more)."""
    if scale is not None:
        s = scale.double().cpu().numpy()[:, None]
        want, size = want / s, size / s
    err = np.abs(_f64(got) - want)
    bound = size * TURN + np.abs(want) * (HALF[dtype] + 2.0**-23) + TINY[dtype]
    assert np.all(err <= bound), float(np.max(err / bound))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t, h, d, pairs", [(1, 1, 64, 32), (7, 5, 128, 64), (600, 3, 64, 16), (513, 2, 80, 20),
                                            (33, 9, 6, 3), (520, 12, 256, 128), (2, 1, 4, 0)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_one_axis(gpu, dtype, t, h, d, pairs, adjacent):
    x, f = _rows(gpu, (t, h, d), dtype, 1), _freq(gpu, pairs)
    pos = torch.arange(t, device=gpu) * 3 + 5
    got = rotary(x, pos, f, interleaved=adjacent, rotary_scale=1.25)
    want, size = oracle.rotate(_f64(x), [pos.cpu().numpy()], f.cpu().numpy(), [pairs], "blocks", adjacent, 1.25)
    _check(got, want, size, dtype)


@pytest.mark.parametrize("order, sections", [("blocks", (16, 24, 24)), ("cycled", (24, 20, 20)), ("blocks", (0, 64)),
                                             ("cycled", (16, 16, 16, 16)), ("cycled", (64, 0, 0)), ("blocks", (1, 62, 1, 0))])
@pytest.mark.parametrize("t", [3, 700])
def test_axes(gpu, order, sections, t):
    x, f = _rows(gpu, (t, 4, 128), torch.bfloat16, 2), _freq(gpu, 64)
    g = torch.Generator(device=gpu).manual_seed(3)
    pos = torch.randint(0, 5000, (len(sections), t), generator=g, device=gpu, dtype=torch.int32)
    got = rotary(x, pos, f, sections=sections, axis_order=order)
    want, size = oracle.rotate(_f64(x), pos.cpu().numpy(), f.cpu().numpy(), sections, order)
    _check(got, want, size, torch.bfloat16)


def test_far_and_negative_positions(gpu):
    pos = torch.tensor([0, -1, 1, 999_999_937, 2**31 - 1, -(2**31)], device=gpu)
    x, f = _rows(gpu, (6, 2, 64), torch.float32, 4), _freq(gpu, 32)
    want, size = oracle.rotate(_f64(x), [pos.cpu().numpy()], f.cpu().numpy(), [32])
    # the float64 products themselves: 2^-53 of an angle of 2^31, on both sides
    for p in (pos, pos.to(torch.int32)):
        _check(rotary(x, p, f), want, size * (1 + 4 * 2.0**31 * 2.0**-53 / TURN), torch.float32)


def test_positions_past_32_bits(gpu):
    """The float64 turns are off by three roundings (the product, 1 / (2 pi) and its product); frequencies
    that are powers of two leave the oracle's own product exact."""
    pos = torch.tensor([2**33 + 1, 2**40 - 3, -(2**45) + 7, 2**52 - 1], device=gpu)
    x, f = _rows(gpu, (4, 2, 64), torch.float32, 6), (0.5 ** torch.arange(32, dtype=torch.float64)).float().to(gpu)
    want, size = oracle.rotate(_f64(x), [pos.cpu().numpy()], f.cpu().numpy(), [32])
    angle = np.abs(pos.cpu().numpy()[:, None].astype(np.float64) * np.tile(f.cpu().numpy(), 2))[:, None]
    _check(rotary(x, pos, f), want, size * (1 + angle * 3 * 2.0**-53 / TURN), torch.float32)


def test_strides_in_place_and_zero_rows(gpu):
    f, pos = _freq(gpu, 24), torch.arange(40, device=gpu)
    big = _rows(gpu, (2, 60, 5, 130), torch.float16, 5)
    x = big[0, 10:50, :, 1:129:2]  # every second channel, from an odd one
    want, size = oracle.rotate(_f64(x), [pos.cpu().numpy()], f.cpu().numpy(), [24])
    before = big.clone()
    out = torch.zeros(64, 40, 5, dtype=torch.float16, device=gpu).permute(1, 2, 0)
    assert rotary(x, pos, f, out=out) is out
    _check(out, want, size, torch.float16)
    assert torch.equal(big, before)
    rotary(x, pos, f, out=x)
    _check(x, want, size, torch.float16)
    before[0, 10:50, :, 1:129:2] = x
    assert torch.equal(big, before)
    assert rotary(x[:0], pos[:0], f).shape == (0, 5, 64)


def _caches(gpu, nb, bs, h, d, dtype, layout):
    if layout == "odd":
        pair = [torch.zeros(bs, h, nb, 2 * d, dtype=dtype, device=gpu)[..., ::2].permute(2, 0, 1, 3) for _ in range(2)]
    else:
        pair = L.alloc_kv_cache(nb, bs, h, d, dtype, gpu, layout)
    for c in pair:
        _raw(c).fill_(3)
    return pair


def _raw(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


@pytest.mark.parametrize("kv", [torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("q", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["paired", "native", "token_major", "odd"])
@pytest.mark.parametrize("t, bs, d", [(5, 16, 64), (531, 16, 128), (600, 8, 40), (520, 16, 256)])
def test_cache_write(gpu, kv, q, layout, t, bs, d):
    """Runs of slots that begin inside a block, jump, and leave the cache; rows of no slot are left as they were."""
    hq, h, pairs = 6, 2, d // 2
    nb = t // bs + 9
    slots = torch.arange(t) + 5
    slots[t // 2:] += 2 * bs + 3  # the second half elsewhere
    slots[1], slots[3] = -1, nb * bs
    if t > 500:
        slots[40:44] = torch.tensor([43, 42, 41, 40]) + 5  # backwards
    dest = slots.to(torch.int32 if t == 531 else torch.int64).to(gpu)
    qn, kn, vn = (_rows(gpu, (t, n, d), q, 6 + i) for i, n in enumerate((hq, h, h)))
    f, pos = _freq(gpu, pairs), torch.randint(0, 9999, (3, t), generator=torch.Generator().manual_seed(1))
    sec = (pairs - 2 * (pairs // 4), pairs // 4, pairs // 4)
    kc, vc = _caches(gpu, nb, bs, h, d, kv, layout)
    ks = vs = None
    if kv == torch.float8_e4m3fn:
        ks, vs = torch.tensor([0.02, 0.03], device=gpu), torch.tensor([0.025, 0.04], device=gpu)
    out = rotary_cache_write(qn, kn, vn, pos.to(gpu), f, dest, kc, vc, sections=sec, k_scale=ks, v_scale=vs)
    want, size = oracle.rotate(_f64(qn), pos.numpy(), f.cpu().numpy(), sec)
    _check(out, want, size, q)
    live = (slots >= 0) & (slots < nb * bs)
    at = slots[live]
    want, size = oracle.rotate(_f64(kn), pos.numpy(), f.cpu().numpy(), sec)
    _check(kc[at // bs, at % bs], want[live.numpy()], size[live.numpy()], kv, ks)
    want = _f64(vn)[live.numpy()]
    if kv == torch.float8_e4m3fn:  # the codes of the framework's own writes
        codes = (vn.float() / vs[:, None])[live.to(gpu)].to(kv)
        assert torch.equal(_raw(vc)[at // bs, at % bs], _raw(codes))
    else:
        assert torch.equal(_raw(vc)[at // bs, at % bs], _raw(vn.to(kv))[live.to(gpu)])
    rest = torch.ones(nb, bs, dtype=torch.bool)
    rest[at // bs, at % bs] = False
    for c in (kc, vc):
        assert bool((_raw(c)[rest.to(gpu)] == 3).all())


def test_nan_and_infinities_stay_in_their_pairs(gpu):
    x = _rows(gpu, (2, 1, 16), torch.float32, 8)
    x[0, 0, 3], x[1, 0, 12] = float("nan"), float("inf")
    got = rotary(x, torch.tensor([7, 9], device=gpu), _freq(gpu, 8))
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[0, 0, [3, 11]] = want[1, 0, [4, 12]] = True
    assert torch.equal(bad, want)
