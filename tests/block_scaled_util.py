"""Plain restatements of the block-scaled cache operators for their tests: float32 steps for the
codes (which are compared bit for bit), float64 for attention."""

from __future__ import annotations

import math

import torch

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
LEAST = 2.0**-40


def least_scale(amax: float, dtype: torch.dtype) -> float:
    """The least scale of values up to amax (float32 arithmetic), NaN where they are not finite."""
    if not math.isfinite(amax):
        return math.nan
    a = torch.tensor(amax, dtype=torch.float32) * (torch.ones(()) / torch.tensor(MOST[dtype], dtype=torch.float32))
    if dtype == torch.int8:
        return max(float(a), LEAST)
    frac, exp = math.frexp(max(float(a), LEAST))
    return math.ldexp(1.0, exp - 1 if frac == 0.5 else exp)


def encode(x: torch.Tensor, scale, dtype: torch.dtype) -> torch.Tensor:
    q = x.float() / torch.as_tensor(scale, dtype=torch.float32)
    if dtype == torch.int8:
        return torch.where(q.isnan(), 0.0, q.clamp(-127, 127).round()).to(torch.int8)
    return q.to(dtype)


def code_bytes(c: torch.Tensor) -> torch.Tensor:
    return c.contiguous().view(torch.uint8)


def write_ref(new, tables, lens, start, codes, scales, bs):
    """One tensor's rows, in place, on the CPU: new [T, H, D], codes [NB, bs, H, D], scales [NB, H]."""
    dtype, nb, heads = codes.dtype, codes.shape[0], codes.shape[2]
    for n in range(len(lens)):
        a, b = (n, n + 1 if lens[n] > 0 else n) if start is None else (start[n], start[n + 1])
        before = lens[n] - (b - a)
        blocks = {}
        for i in range(a, b):
            pos = before + i - a
            if 0 <= pos < len(tables[n]) * bs and 0 <= tables[n][pos // bs] < nb:
                blocks.setdefault(pos // bs, []).append((pos % bs, i))
        for j, rows in blocks.items():
            blk, first = tables[n][j], rows[0][0]
            for h in range(heads):
                x = torch.stack([new[i, h].float() for _, i in rows])
                m = x.abs().max()
                need = least_scale(math.nan if bool(x.isnan().any()) else float(m), dtype)
                old = float(scales[blk, h]) if first > 0 else 0.0
                s = math.nan if math.isnan(old) or math.isnan(need) else max(old, need)
                if first > 0 and s != old:
                    was = codes[blk, :first, h].float() * torch.tensor(old, dtype=torch.float32)
                    codes[blk, :first, h] = encode(was, s, dtype)
                for k, (off, _) in enumerate(rows):
                    codes[blk, off, h] = encode(x[k], s, dtype)
                scales[blk, h] = s


def filled(nb, bs, heads, dim, dtype, gen, spread=1.0):
    """Random codes [NB, bs, H, D] with their scales [NB, H], a block's largest value reached."""
    x = torch.randn(nb, bs, heads, dim, generator=gen) * torch.exp2(spread * torch.randn(nb, 1, heads, 1, generator=gen))
    s = torch.tensor([[least_scale(float(x[b, :, h].abs().max()), dtype) for h in range(heads)] for b in range(nb)])
    return encode(x, s[:, None, :, None], dtype), s.reshape(nb, heads)


def dense(codes, scales, table, n, bs):
    """[H, n, D] float64 values of a table's first n tokens; tokens of blocks outside the cache None-marked by `ok`."""
    nb = codes.shape[0]
    ids = torch.tensor([table[t // bs] for t in range(n)], dtype=torch.long)
    ok = (ids >= 0) & (ids < nb)
    ids = ids.clamp(0, nb - 1)
    x = codes[ids, torch.arange(n) % bs].float().double() * scales[ids].double()[..., None]
    return x.transpose(0, 1), ok


def attend_ref(q, k_codes, k_scales, v_codes, v_scales, table, n, scale, bs=16):
    """One query row [Hq, D] over a sequence's first n tokens, in float64: (output, sum of p |v|, largest sum of
    |q k| of a score, sum of |v|)."""
    hq, d = q.shape
    hkv = k_codes.shape[2]
    g = hq // hkv
    n = min(n, len(table) * bs)
    if n <= 0:
        return torch.zeros(hq, d).double(), torch.zeros(hq, d).double(), 0.0, torch.zeros(hq, d).double()
    (k, ok), (v, _) = dense(k_codes, k_scales, table, n, bs), dense(v_codes, v_scales, table, n, bs)
    k, v, idx = k[:, ok], v[:, ok], torch.arange(hq) // g
    if not bool(ok.any()):
        return torch.zeros(hq, d).double(), torch.zeros(hq, d).double(), 0.0, torch.zeros(hq, d).double()
    qd = q.double()
    s = (qd[:, None] * k[idx]).sum(-1) * scale
    size = float(((qd.abs()[:, None] * k[idx].abs()).sum(-1) * abs(scale)).max())
    p = torch.softmax(s, -1)
    return (p[..., None] * v[idx]).sum(1), (p[..., None] * v[idx].abs()).sum(1), size, v[idx].abs().sum(1)


def assert_attended(got, refs, out_dtype, dim, tokens, p_round, what, p_least=0.0):
    """Every element within what the kernels' roundings can add up to: the output's own half step; of the sum of
    p |v|, the rounding of p ahead of the product with V (p_round), float32 sums over the tokens (one rounding a
    tile of 32 and its tree of 5), and what an error of a score does to every weight, twice (numerator and sum): a
    score is a float32 sum of dim / 32 + 5 roundings of terms of `size` in all, times a factor (2 roundings), and
    its exponential is good to 2^-21.

    p_least: the absolute rounding of a small weight.  In fp16 it is half of the smallest step, 2^-25, where p is
    below 2^-14; p is relative to a reference that is at most the row's largest score, so the sum of all is 1 or
    more, and a token's |v| enters the output by at most 2^-25 too much or too little."""
    ref = torch.stack([r[0] for r in refs])
    size = max(r[2] for r in refs)
    weight = 2.0 * (size * (dim / 32 + 7) * 2.0**-23 + 2.0**-21)
    per = p_round + (tokens / 32 + 6) * 2.0**-23 + weight
    tol = torch.finfo(out_dtype).eps / 2 * ref.abs() * (1 + per) + per * torch.stack([r[1] for r in refs])
    tol = tol + p_least * torch.stack([r[3] for r in refs])
    # (results below the smallest normal number are rounded to its last bit)
    tol = tol + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
    err = (got.double().cpu() - ref).abs()
    worst = float((err / tol.clamp(min=1e-300)).max()) if err.numel() else 0.0
    print(f"[parity] {what} worst error / bound {worst:.3f}", flush=True)
    assert bool((err <= tol).all()), (what, worst)
