"""Operators of a bounded KV cache: rows enter it rotated, are attended with their weights
accumulated, and leave by those weights.

  rotary   `rotary_cache_write`: rotary positions of one or several axes on the queries and keys
           of new tokens, keys and values written to their paged slots
  decode   `paged_attention_weights`: decode attention of one new token a sequence that also adds
           every cached token's attention weight to the sequence's account
  chunk    `chunk_attention_weights`: the same account for the rows of prompts and chunks
  select   `evict_select`: which tokens each head keeps, from the accounts
  move     `evict_move`: the kept tokens' rows, weights and positions moved into the holes

Head shapes are those of this repository's workloads; K and V are N(0, 1), in FP8 caches as codes
under per-KV-head scales.  Lengths come from the case itself ("sizes" seeds them), values and block
placement from the seed.
"""

from __future__ import annotations

import importlib
import math
import random
import sys
from pathlib import Path

import torch

own = False

BS = 16  # tokens per block

# query heads, KV heads, head_dim
HEADS = {
    "opt125m": (12, 12, 64),
    "tinyllama": (32, 4, 64),
    "llama3_8b": (32, 8, 128),
    "llama3_70b": (64, 8, 128),
}
DTYPES = {
    "float32": torch.float32,
    "float16": torch.float16,
    "bfloat16": torch.bfloat16,
    "float8_e4m3fn": torch.float8_e4m3fn,
}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2, "float8_e4m3fn": 1}


_ENTRY = {}  # the framework's entry points, imported once as a user's program does


def _entry(module, name):
    if own and name not in _ENTRY:
        at = str(Path(__file__).resolve().parent.parent / "llm-compileforge_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        _ENTRY[name] = getattr(importlib.import_module(module), name)
    return _ENTRY[name]


def _rotary(name, heads, q, kv, batch, lo, hi, **more):
    return {"name": name, "kind": "rotary", "heads": heads, "q": q, "kv": kv, "batch": batch, "lo": lo, "hi": hi,
            "axes": 3, "order": "blocks", "pairs": "halves", "part": 1.0, "first": 0, "layout": "paired", "sizes": 0,
            **more}


def _decode(name, heads, q, kv, batch, lo, hi, **more):
    return {"name": name, "kind": "decode", "heads": heads, "q": q, "kv": kv, "batch": batch, "lo": lo, "hi": hi,
            "shared": 0, "per_head": True, "decay": 1.0, "layout": "paired", "sizes": 0, **more}


def _chunk(name, heads, q, kv, chunks, rows_lo, rows_hi, lo, hi, **more):
    return {"name": name, "kind": "chunk", "heads": heads, "q": q, "kv": kv, "chunks": chunks, "rows_lo": rows_lo,
            "rows_hi": rows_hi, "lo": lo, "hi": hi, "observe": 0, "per_head": True, "decay": 1.0, "layout": "paired",
            "sizes": 0, **more}


def _evict(name, kind, heads, batch, lo, hi, budget, **more):
    return {"name": name, "kind": kind, "heads": heads, "kv": "bfloat16", "batch": batch, "lo": lo, "hi": hi,
            "budget": budget, "sink": 4, "recent": budget // 8, "moved_before": True, "per_head": True,
            "layout": "paired", "sizes": 0, **more}


def listed():
    return [
        # the smallest call: a decode step's 32 new tokens, a multimodal model's three axes
        _rotary("rotary_step_tinyllama_bf16", "tinyllama", "bfloat16", "bfloat16", 32, 1, 1, first=700),
        # four prompts' rows into an FP8 cache
        _rotary("rotary_prompt_llama3_8b_fp8", "llama3_8b", "bfloat16", "float8_e4m3fn", 4, 700, 2000, order="cycled",
                sizes=1),
        # text far into a long context in float32, adjacent pairs, half of the channels, the reference's own layout
        _rotary("rotary_far_opt125m_f32", "opt125m", "float32", "float32", 1, 1237, 1237, axes=1, pairs="adjacent",
                part=0.5, first=1000000, layout="token_major", sizes=2),
        # four requests of a small float32 model
        _decode("weights_opt125m_f32", "opt125m", "float32", "float32", 4, 128, 512, sizes=3),
        # a serving batch over an FP8 cache, half of it on a radix-shared prefix
        _decode("weights_llama3_8b_fp8", "llama3_8b", "bfloat16", "float8_e4m3fn", 64, 1024, 8192, shared=1024,
                sizes=4),
        # one user with a long context, one account for all heads, older steps fading
        _decode("weights_one_long_bf16", "llama3_8b", "bfloat16", "bfloat16", 1, 29999, 29999, per_head=False,
                decay=0.95, sizes=5),
        # whole prompts, every row counted
        _chunk("chunk_prompt_tinyllama_bf16", "tinyllama", "bfloat16", "bfloat16", 2, 1500, 4000, 0, 0,
               layout="token_major", sizes=6),
        # the last chunk of long prompts, its last 64 rows as observers
        _chunk("chunk_observe_llama3_8b_fp8", "llama3_8b", "bfloat16", "float8_e4m3fn", 4, 512, 512, 4000, 12000,
               observe=64, sizes=7),
        # a decode batch that has grown one block past its budget
        _evict("select_step_llama3_8b", "select", "llama3_8b", 64, 2049, 2064, 2048, sizes=8),
        # prompts cut to their budget
        _evict("select_prompt_llama3_8b", "select", "llama3_8b", 4, 20000, 30000, 4096, moved_before=False, sizes=9),
        _evict("move_step_llama3_8b_bf16", "move", "llama3_8b", 64, 2049, 2064, 2048, sizes=10),
        _evict("move_prompt_llama3_8b_fp8", "move", "llama3_8b", 4, 20000, 30000, 4096, kv="float8_e4m3fn",
               moved_before=False, sizes=11),
    ]


# ---- drawn cases ----------------------------------------------------------------------

MAX_BYTES = 5.0e8
MAX_F32_BYTES = 1.5e8
MAX_PLAIN = 6.0e8  # scores or cached values that the plain form holds at once


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw_one(rng)
        del case["name"]
        most = MAX_F32_BYTES if "float32" in (case.get("q"), case["kv"]) else MAX_BYTES
        if work(case)["bytes"] <= most and _plain_size(case) <= MAX_PLAIN:
            return case


def _types(rng, f32):
    pairs = [("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float8_e4m3fn"),
             ("float16", "float8_e4m3fn")]
    return rng.choice(pairs + ([("float32", "float32"), ("float32", "bfloat16")] if f32 else []))


def _draw_one(rng):
    kind = rng.choice(["rotary", "rotary", "decode", "decode", "decode", "chunk", "chunk", "select", "move"])
    heads = rng.choice(list(HEADS))
    layout = rng.choice(["paired", "paired", "native", "token_major"])
    sizes = rng.randrange(1 << 30)
    if kind == "rotary":
        q, kv = _types(rng, True)
        batch = _log(rng, 1, 128)
        lo = rng.choice([1, _log(rng, 2, 2048)])
        return _rotary("", heads, q, kv, batch, lo, lo if lo == 1 else _log(rng, lo, 4 * lo), axes=rng.choice([1, 2, 3, 3]),
                       order=rng.choice(["blocks", "cycled"]), pairs=rng.choice(["halves", "halves", "adjacent"]),
                       part=rng.choice([1.0, 1.0, 0.5]), first=_log(rng, 1, 1000000), layout=layout, sizes=sizes)
    if kind == "decode":
        q, kv = _types(rng, True)
        lo = _log(rng, 16, 8192)
        return _decode("", heads, q, kv, _log(rng, 1, 128), lo, min(32768, _log(rng, lo, 4 * lo)),
                       shared=BS * rng.randint(1, lo // BS) if rng.random() < 0.25 else 0,
                       per_head=rng.random() < 0.7, decay=rng.choice([1.0, 1.0, 0.9, 0.0]), layout=layout, sizes=sizes)
    if kind == "chunk":
        q, kv = _types(rng, False)
        rows = _log(rng, 2, 4000)
        cached = rng.choice([0, _log(rng, 16, 12000)])
        return _chunk("", heads, q, kv, _log(rng, 1, 8), max(1, rows // 2), rows, cached // 2, cached,
                      observe=rng.choice([0, 0, _log(rng, 1, 128)]), per_head=rng.random() < 0.7,
                      decay=rng.choice([1.0, 1.0, 0.9, 0.0]), layout=layout, sizes=sizes)
    budget = _log(rng, 16, 8192)
    lo = _log(rng, max(1, budget // 2), 4 * budget)
    return _evict("", kind, heads, _log(rng, 1, 128), lo, min(32768, _log(rng, lo, 4 * lo)), budget,
                  kv=_types(rng, True)[1], sink=rng.choice([0, 1, 4]), recent=rng.randint(0, budget - 4),
                  moved_before=rng.random() < 0.7, per_head=rng.random() < 0.8, layout=layout, sizes=sizes)


def _plain_size(case):
    hq, hkv, d = HEADS[case["heads"]]
    lens = _lens(case)
    if case["kind"] == "decode":
        return len(lens) * max(lens) * hkv * d
    if case["kind"] == "chunk":
        return len(lens) * max(r for r, _ in _chunks(case)) * max(lens) * hq // (8 if case["observe"] else 1)
    if case["kind"] == "rotary":
        return sum(lens) * hq * d
    return len(lens) * max(lens) * hkv * d


# ---- sizes that follow from the case alone ---------------------------------------------


def _chunks(case):
    """(rows, cached tokens) of each chunk."""
    rng = random.Random(case["sizes"] + 1)
    return [(rng.randint(case["rows_lo"], case["rows_hi"]), rng.randint(case["lo"], case["hi"]))
            for _ in range(case["chunks"])]


def _lens(case):
    """Tokens of every sequence (rotary: the new ones)."""
    if case["kind"] == "chunk":
        return [r + c for r, c in _chunks(case)]
    rng = random.Random(case["sizes"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def _blocks(n):
    return -(-n // BS)


def _rotated(case):
    """Rotated pairs of a head, and how many of them each axis has."""
    d = HEADS[case["heads"]][2]
    pairs = int(d * case["part"]) // 2
    a = case["axes"]
    other = pairs // (a + 1) if a > 1 else 0
    return pairs, [pairs - (a - 1) * other] + [other] * (a - 1)


def _visible(rows, cached, observe):
    """(row, token) pairs of a causal chunk's observed rows."""
    n = rows if observe == 0 else min(rows, observe)
    first = cached + rows - n + 1  # tokens that the first observed row sees
    return n * first + n * (n - 1) // 2


def work(case):
    hq, hkv, d = HEADS[case["heads"]]
    kind, kb = case["kind"], BYTES[case["kv"]]
    lens = _lens(case)
    n = sum(lens)
    hw = hkv if case.get("per_head", True) else 1
    if kind == "rotary":
        qb, pairs = BYTES[case["q"]], _rotated(case)[0]
        return {"bytes": n * (2 * hq * d * qb + 2 * hkv * d * (qb + kb) + 4 * case["axes"] + 8),
                "flops": 6.0 * n * (hq + hkv) * pairs}
    if kind == "decode":
        once = n - sum(min(case["shared"], x) for x in lens[1: max(1, len(lens) // 2)]) if len(lens) > 1 else n
        return {"bytes": once * 2 * hkv * d * kb + n * hw * (8 if case["decay"] else 4)
                + 2 * len(lens) * hq * d * BYTES[case["q"]], "flops": 4.0 * n * hq * d}
    if kind == "chunk":
        ch = _chunks(case)
        seen = [min(r, case["observe"] or r) for r, _ in ch]
        return {"bytes": n * hkv * d * kb + n * hw * 8 + sum(seen) * hq * d * BYTES[case["q"]],
                "flops": 2.0 * hq * d * sum(_visible(r, c, case["observe"]) for r, c in ch)}
    slots = len(lens) * case["budget"] * hw
    if kind == "select":
        return {"bytes": n * hw * (8 if case["moved_before"] else 4) + 4 * slots, "flops": 2.0 * n * hw}
    moves = 0.0  # what is kept of the tail: the newest, and its share of the rest
    for x in lens:
        free = case["budget"] - case["sink"] - case["recent"]
        tail = x - case["budget"]
        if tail > 0:
            moves += min(tail, case["recent"]) + free * max(0, tail - case["recent"]) / (
                x - case["sink"] - case["recent"])
    return {"bytes": 4 * slots + moves * hkv * 4 * d * kb + moves * hw * 16, "flops": 1.0 * slots}


# ---- inputs ----------------------------------------------------------------------------


def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _randn(shape, dtype, seed):
    return torch.randn(shape, generator=_gen(seed), device=_dev(), dtype=torch.float32).to(dtype)


def _raw(t):
    """FP8 codes as bytes; anything else as it is."""
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _empty_caches(nb, hkv, d, dtype, layout):
    """K and V as [NB, 16, Hkv, D] views: token rows, or tiles of a (block, head) with V channel-major."""
    if layout == "token_major":
        return tuple(torch.empty(nb, BS, hkv, d, dtype=dtype, device=_dev()) for _ in range(2))
    if layout == "native":
        k = torch.empty(nb, hkv, BS, d, dtype=dtype, device=_dev())
        v = torch.empty(nb, hkv, d, BS, dtype=dtype, device=_dev())
    else:
        both = torch.empty(nb, hkv, 2, BS * d, dtype=dtype, device=_dev())
        k, v = both[:, :, 0].view(nb, hkv, BS, d), both[:, :, 1].view(nb, hkv, d, BS)
    return k.permute(0, 2, 1, 3), v.permute(0, 3, 1, 2)


def _caches(case, nb, seed):
    """Filled caches and, over FP8, their scales."""
    _, hkv, d = HEADS[case["heads"]]
    dtype = DTYPES[case["kv"]]
    pair = _empty_caches(nb, hkv, d, dtype, case["layout"])
    scales = [None, None]
    for i, c in enumerate(pair):
        x = _randn((nb, BS, hkv, d), torch.float32, 10 * seed + 1 + i)
        if dtype == torch.float8_e4m3fn:
            scales[i] = (0.016 + 0.004 * torch.rand(hkv, generator=_gen(10 * seed + 3 + i), device=_dev())).contiguous()
            x = x / scales[i][:, None]
        _raw(c).copy_(_raw(x.to(dtype)))
    return *pair, *scales


def _tables(case, seed):
    """int32 block tables of every sequence, scattered over a pool with some blocks unused; blocks in the pool."""
    lens = [x + case.get("first", 0) % BS for x in _lens(case)] if case["kind"] == "rotary" else _lens(case)
    shared = case.get("shared", 0) // BS if len(lens) > 1 else 0
    n_shared = len(lens) // 2 if shared else 0
    nb = sum(_blocks(n) for n in lens) + shared + 16
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).tolist()
    at, rows = shared, []
    for i, n in enumerate(lens):
        t = perm[:shared][: _blocks(n)] if i < n_shared else []
        take = _blocks(n) - len(t)
        rows.append(t + perm[at: at + take])
        at += take
    width = max(len(t) for t in rows)
    tables = torch.tensor([t + [0] * (width - len(t)) for t in rows], dtype=torch.int32)
    common = [0] + [min(shared * BS, lens[i - 1], lens[i]) if 0 < i < n_shared else 0 for i in range(1, len(lens))]
    return tables, nb, torch.tensor(common, dtype=torch.int32).to(_dev()) if shared else None


def _int32(x):
    return torch.tensor(x, dtype=torch.int32).to(_dev())


def _accounts(case, lens, width, seed):
    """Accounts as eight earlier steps leave them: heavy-tailed, the first tokens heaviest."""
    hq, hkv, _ = HEADS[case["heads"]]
    hw = hkv if case["per_head"] else 1
    w = torch.empty(len(lens), hw, width, device=_dev()).exponential_(generator=_gen(10 * seed + 5)).square_()
    w *= (4.0 * hq / hw) / torch.tensor(lens, dtype=torch.float32).clamp(min=1).to(_dev())[:, None, None]
    w[:, :, :2] *= 50.0
    return w


def prepare(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    lens = _lens(case)
    tables, nb, common = _tables(case, seed)
    s = dict(case, lens=_int32(lens), tables=tables.to(_dev()), scale=1.0 / math.sqrt(d), common=common, top=max(lens))
    if case["kind"] != "select":
        s["k"], s["v"], s["ks"], s["vs"] = _caches(case, nb, seed)
    if case["kind"] == "rotary":
        return _prepare_rotary(s, tables, lens, seed)
    width = tables.shape[1] * BS
    if case["kind"] in ("decode", "chunk"):
        rows = len(lens) if case["kind"] == "decode" else sum(r for r, _ in _chunks(case))
        s["q"] = _randn((rows, hq, d), DTYPES[case["q"]], 10 * seed + 6)
        s["w"] = _accounts(case, lens, width, seed)
    if case["kind"] == "chunk":
        starts = [0]
        for r, _ in _chunks(case):
            starts.append(starts[-1] + r)
        s["start"], s["rows"] = _int32(starts), max(min(r, case["observe"] or r) for r, _ in _chunks(case))
    if case["kind"] in ("select", "move"):
        s["w"] = _accounts(case, lens, width, seed)
        s["pos"] = s["kept"] = s["seen"] = None
        if case["moved_before"]:  # the budget's tokens in any order, of a sequence three times as long
            s["seen"] = 3 * s["lens"]
            s["kept"] = s["lens"].clamp(max=case["budget"])
            key = torch.rand(s["w"].shape, generator=_gen(10 * seed + 7), device=_dev())
            at = torch.arange(width, device=_dev())
            key[(at >= s["kept"][:, None]).unsqueeze(1).expand_as(key)] = 2.0
            order = key.argsort(-1).argsort(-1)  # a permutation of the kept slots
            s["pos"] = (order * 2).to(torch.int32).contiguous()
    if case["kind"] == "move":
        s["keep"] = _select(s)[0]
    return s


def _prepare_rotary(s, tables, lens, seed):
    hq, hkv, d = HEADS[s["heads"]]
    n, pairs = sum(lens), _rotated(s)[0]
    dtype = DTYPES[s["q"]]
    s["q"], s["k_new"], s["v_new"] = (_randn((n, h, d), dtype, 10 * seed + 5 + i) for i, h in enumerate((hq, hkv, hkv)))
    s["inv_freq"] = (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().to(_dev())
    off = s["first"] % BS  # the first new row's place in its block
    seq = torch.repeat_interleave(torch.tensor(lens))
    at = off + torch.cat([torch.arange(x) for x in lens])
    s["slots"] = (tables[seq, at // BS].long() * BS + at % BS).to(_dev())
    text = torch.cat([torch.arange(x) for x in lens]) + s["first"]
    # text runs along all axes; every other stretch of 256 rows is an image of 16 x 16
    image = (torch.arange(n) // 256) % 2 == 1
    at = torch.arange(n)
    axes = [torch.where(image, text - at % 256, text), torch.where(image, text - at % 256 + at % 256 // 16, text),
            torch.where(image, text - at % 256 + at % 16, text)]
    s["positions"] = torch.stack(axes[: s["axes"]]).to(torch.int32).to(_dev())
    s["n_axes"], s["sections"] = s["axes"], tuple(_rotated(s)[1])
    return s


# ---- the plain forms -------------------------------------------------------------------


def _axis_of_pair(s):
    pairs, a = sum(s["sections"]), s["n_axes"]
    j = torch.arange(pairs, device=_dev())
    if s["order"] == "cycled":
        return torch.where((j % a > 0) & (j < a * s["sections"][-1]), j % a, 0)
    edges = torch.tensor(s["sections"], device=_dev()).cumsum(0)
    return (j[:, None] >= edges).sum(1)


def _turn(x, cos, sin, adjacent):
    pairs = cos.shape[-1]
    x = x.float()
    if adjacent:
        a, b = x[..., 0: 2 * pairs: 2], x[..., 1: 2 * pairs: 2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs: 2 * pairs]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * pairs:]), -1)


def _put(cache, slots, rows, scale):
    if scale is not None:
        rows = rows / scale[:, None]
    _raw(cache)[slots // BS, slots % BS] = _raw(rows.to(cache.dtype))


def _run_rotary(s):
    # angles of far positions in 64 bits
    angle = s["positions"].double()[_axis_of_pair(s)].T * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    adjacent = s["pairs"] == "adjacent"
    q = _turn(s["q"], cos, sin, adjacent).to(s["q"].dtype)
    _put(s["k"], s["slots"], _turn(s["k_new"], cos, sin, adjacent), s["ks"])
    _put(s["v"], s["slots"], s["v_new"].float(), s["vs"])
    return [q, s["k"], s["v"]]


def _dense(cache, tables, scale, top):
    """[B, Hkv, top, D] float32 values of the tables' tokens."""
    at = torch.arange(top, device=_dev())
    x = cache[tables[:, at // BS].long(), at % BS] if cache.dtype != torch.float8_e4m3fn else _raw(cache)[
        tables[:, at // BS].long(), at % BS].view(torch.float8_e4m3fn)
    x = x.float()
    return (x if scale is None else x * scale[:, None]).transpose(1, 2).contiguous()


def _account(s, p, fresh, live):
    """New accounts from the weights p [B, Hkv, rows, tokens] (rows: query rows and heads)."""
    top = p.shape[-1]
    add = p.sum(2)
    if not s["per_head"]:
        add = add.sum(1, keepdim=True)
    old = s["w"][:, :, :top]
    base = torch.where(fresh[:, None], 0.0, old * s["decay"] if s["decay"] else torch.zeros_like(old))
    s["w"][:, :, :top] = torch.where(live[:, None], base + add, old)


def _run_decode(s):
    b, hq, d = s["q"].shape
    k, v = _dense(s["k"], s["tables"], s["ks"], s["top"]), _dense(s["v"], s["tables"], s["vs"], s["top"])
    hkv = k.shape[1]
    q = s["q"].float().view(b, hkv, hq // hkv, d)
    at = torch.arange(s["top"], device=_dev())
    live = at < s["lens"][:, None]
    sc = (q @ k.transpose(-1, -2).contiguous()) * s["scale"]
    sc = torch.where(live[:, None, None], sc, -math.inf)
    p = (sc - sc.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = (p @ v).reshape(b, hq, d).to(s["q"].dtype)
    _account(s, p, at == s["lens"][:, None] - 1, live)
    return [out, s["w"]]


def _run_chunk(s):
    k = _dense(s["k"], s["tables"], s["ks"], s["top"])
    n, hkv, _, d = k.shape
    hq = s["q"].shape[1]
    # the last observed row of a chunk last; rows before a short chunk's first are masked
    i = torch.arange(s["rows"], device=_dev()) - s["rows"]
    size = (s["start"][1:] - s["start"][:-1])[:, None]
    counted = -i <= (size.clamp(max=s["observe"]) if s["observe"] else size)
    q = s["q"][(s["start"][1:, None] + i).clamp(min=0).long()].float()
    q = q.view(n, s["rows"], hkv, hq // hkv, d).transpose(1, 2).reshape(n, hkv, -1, d)
    at = torch.arange(s["top"], device=_dev())
    sees = (at <= (s["lens"][:, None] + i)[..., None]) & counted[..., None]  # [n, rows, tokens]
    sc = (q @ k.transpose(-1, -2).contiguous()).mul_(s["scale"]).view(n, hkv, s["rows"], hq // hkv, -1)
    sc.masked_fill_(~sees[:, None, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True).clamp(min=-1e30)
    sc.sub_(top).exp_()
    sc.div_(sc.sum(-1, keepdim=True).clamp(min=1e-30))
    live = at < s["lens"][:, None]
    _account(s, sc.flatten(2, 3), live & (at >= s["lens"][:, None] - size), live)
    return [s["w"]]


def _select(s):
    """(keep, new lengths): per head the protected tokens, then the heaviest."""
    w, lens, budget = s["w"], s["lens"][:, None, None].long(), s["budget"]
    width = w.shape[-1]
    at = torch.arange(width, device=_dev())
    live = at < lens
    if s["pos"] is None:
        pos, seen = at.expand_as(w), lens
    else:
        seen = s["seen"][:, None, None].long()
        pos = torch.where(at < s["kept"][:, None, None], s["pos"].long(), seen - lens + at)
    safe = live & ((pos < s["sink"]) | (pos >= seen - s["recent"]))
    bits = (w + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -2147483648 - bits, bits)
    key = torch.where(safe, 1 << 33, torch.where(live, key, -(1 << 33))) * (1 << 20) - at
    size = lens.clamp(max=budget)
    rank = key.argsort(-1, descending=True).argsort(-1)
    kept = live & (rank < budget)
    hole, mover = ~kept & (at < size), kept & (at >= size)
    # the k-th mover's index, for the k-th hole
    order = torch.where(mover, at, width + at).argsort(-1)
    turn = (hole.long().cumsum(-1) - 1).clamp(min=0)
    keep = torch.where(hole, order.gather(-1, turn), at)
    keep = torch.where(at < size, keep, -1)[..., :budget]
    keep = torch.nn.functional.pad(keep, (0, budget - keep.shape[-1]), value=-1)
    return keep.to(torch.int32).contiguous(), size.view(-1).to(torch.int32)


def _rows_to(cache, blk, off, head, src_blk, src_off):
    raw = _raw(cache)
    raw[blk, off, head] = raw[src_blk, src_off, head]


def _run_move(s):
    keep = s["keep"].long()
    b, hw, budget = keep.shape
    at = torch.arange(budget, device=_dev())
    if s["pos"] is not None:
        source = keep.clamp(min=0)
        first = (s["seen"] - s["lens"])[:, None, None].long()
        n = min(budget, s["pos"].shape[-1])
        pos = torch.where(source < s["kept"][:, None, None], s["pos"].long().gather(-1, source), first + source)[..., :n]
        s["pos"][..., :n] = torch.where(keep[..., :n] >= 0, pos.to(torch.int32), s["pos"][..., :n])
    seq, head, slot = ((keep >= 0) & (keep != at)).nonzero(as_tuple=True)
    source = keep[seq, head, slot]
    s["w"][seq, head, slot] = s["w"][seq, head, source]
    heads = head if hw > 1 else torch.arange(s["k"].shape[2], device=_dev())[:, None]
    blk, src_blk = s["tables"][seq, slot // BS].long(), s["tables"][seq, source // BS].long()
    _rows_to(s["k"], blk, slot % BS, heads, src_blk, source % BS)
    _rows_to(s["v"], blk, slot % BS, heads, src_blk, source % BS)
    return [s["k"], s["v"], s["w"]] + ([] if s["pos"] is None else [s["pos"]])


# ---- one pass --------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "rotary":
        return _run_rotary(s)
    if s["kind"] == "decode":
        return _run_decode(s)
    if s["kind"] == "chunk":
        return _run_chunk(s)
    if s["kind"] == "select":
        return list(_select(s))
    return _run_move(s)


def _run_own(s):
    if own:
        if s["kind"] == "rotary":
            q = _entry("kernels.rotary", "rotary_cache_write")(
                s["q"], s["k_new"], s["v_new"], s["positions"], s["inv_freq"], s["slots"], s["k"], s["v"],
                sections=s["sections"], axis_order=s["order"], interleaved=s["pairs"] == "adjacent", k_scale=s["ks"],
                v_scale=s["vs"])
            return [q, s["k"], s["v"]]
        if s["kind"] == "decode":
            out = _entry("kernels.paged_attention", "paged_attention_weights")(
                s["q"], s["k"], s["v"], s["tables"], s["lens"], s["w"], BS, s["scale"], decay=s["decay"],
                k_scale=s["ks"], v_scale=s["vs"], shared_prefix_lens=s["common"])
            return [out, s["w"]]
        if s["kind"] == "chunk":
            _entry("kernels.paged_attention", "chunk_attention_weights")(
                s["q"], s["k"], s["tables"], s["lens"], s["start"], s["w"], BS, s["scale"], decay=s["decay"],
                observe=s["observe"], k_scale=s["ks"])
            return [s["w"]]
        if s["kind"] == "select":
            return list(_entry("kernels.kv_eviction", "evict_select")(
                s["w"], s["lens"], s["budget"], sink=s["sink"], recent=s["recent"], positions=s["pos"], kept=s["kept"],
                seen=s["seen"]))
        _entry("kernels.kv_eviction", "evict_move")(
            s["keep"], s["lens"], s["tables"], s["k"], s["v"], weights=s["w"], positions=s["pos"], kept=s["kept"],
            seen=s["seen"])
        return [s["k"], s["v"], s["w"]] + ([] if s["pos"] is None else [s["pos"]])


# ---- from the definitions, in 64 bits --------------------------------------------------


def _tokens(cache, table, n, h, scale):
    """Head h's first n token rows [n, D] of one sequence, in float64."""
    blocks = _raw(cache)[table[: _blocks(n)].long(), :, h]
    if cache.dtype == torch.float8_e4m3fn:
        blocks = blocks.contiguous().view(torch.float8_e4m3fn).float()
    x = blocks.double().reshape(-1, cache.shape[3])[:n]
    return x if scale is None else x * scale[h].double()


def _softmax64(q, k, scale, last):
    """Weights of rows q [rows, D] over tokens k, row i seeing the tokens up to last[i]."""
    e = (k @ q.T.contiguous()).T * scale
    e[torch.arange(k.shape[0], device=_dev())[None] > last[:, None]] = -math.inf
    e = torch.exp(e - e.max(1, keepdim=True).values)
    return e / e.sum(1, keepdim=True)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(s)
    if case["kind"] == "select":
        return None  # whole numbers
    if case["kind"] == "move":
        return _exact_move(s)
    hq, hkv, d = HEADS[case["heads"]]
    g, hw = hq // hkv, s["w"].shape[1]
    w = s["w"].double()
    out = None if case["kind"] == "chunk" else torch.zeros(s["q"].shape, dtype=torch.float64, device=_dev())
    starts = None if case["kind"] == "decode" else s["start"].tolist()
    for b, n in enumerate(_lens(case)):
        rows = 1 if starts is None else starts[b + 1] - starts[b]
        seen = min(rows, case.get("observe") or rows)
        begin = b if starts is None else starts[b + 1] - seen
        last = torch.arange(n - seen, n, device=_dev())
        w[b, :, : n - rows] *= case["decay"]
        w[b, :, n - rows: n] = 0.0
        for h in range(hkv):
            k = _tokens(s["k"], s["tables"][b], n, h, s["ks"])
            for j in range(h * g, h * g + g):
                p = _softmax64(s["q"][begin: begin + seen, j].double(), k, s["scale"], last)
                w[b, h if hw > 1 else 0, :n] += p.sum(0)
                if out is not None:
                    out[b, j] = (p @ _tokens(s["v"], s["tables"][b], n, h, s["vs"]))[0]
    return [w] if out is None else [out, w]


def _exact_rotary(s):
    pairs = s["inv_freq"].numel()
    if s["order"] == "cycled":
        axis = [j % s["n_axes"] if j % s["n_axes"] and j < s["n_axes"] * s["sections"][j % s["n_axes"]] else 0
                for j in range(pairs)]
    else:
        axis = [a for a, c in enumerate(s["sections"]) for _ in range(c)]
    first = [j if s["pairs"] == "halves" else 2 * j for j in range(pairs)]
    second = [j + (pairs if s["pairs"] == "halves" else 1) for j in first]
    unit = torch.polar(torch.ones((), dtype=torch.float64, device=_dev()),
                       s["positions"][axis].double() * s["inv_freq"].double()[:, None]).T[:, None]
    got = []
    for x in (s["q"], s["k_new"]):
        x = x.double()
        z = torch.complex(x[..., first], x[..., second]) * unit
        x[..., first], x[..., second] = z.real, z.imag
        got.append(x)
    outs = [got[0]]
    for cache, rows, scale in ((s["k"], got[1], s["ks"]), (s["v"], s["v_new"].double(), s["vs"])):
        whole = cache.float().double().contiguous() if cache.dtype == torch.float8_e4m3fn else cache.double().contiguous()
        whole.view(-1, *whole.shape[2:])[s["slots"]] = rows if scale is None else rows / scale.double()[:, None]
        outs.append(whole)
    return outs


def _exact_move(s):
    """Every slot's values from its source, one sequence and head at a time."""
    caches = [(_raw(c).contiguous().view(c.dtype) if c.dtype == torch.float8_e4m3fn else c.contiguous()).float().double()
              for c in (s["k"], s["v"])]
    w = s["w"].double()
    for b in range(s["keep"].shape[0]):
        table = s["tables"][b].long()
        slots = (table[:, None] * BS + torch.arange(BS, device=_dev())).flatten()
        for h in range(s["keep"].shape[1]):
            keep = s["keep"][b, h][s["keep"][b, h] >= 0].long()
            w[b, h, : keep.numel()] = w[b, h][keep]
            heads = slice(h, h + 1) if s["keep"].shape[1] > 1 else slice(None)
            for c in caches:
                flat = c.view(-1, *c.shape[2:])[:, heads]
                flat[slots[: keep.numel()]] = flat[slots[keep]]
    return caches + [w] + ([] if s["pos"] is None else [None])
