"""Accounts of prompt chunks without a GPU: refusals and the workspace."""

from __future__ import annotations

import pytest
import torch

from cf_hip import _abi, ops
from kernels.paged_attention import chunk_attention_weights
from python_runtime.engine.cache_manager import CacheManager


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="ROCm"):
        chunk_attention_weights(torch.zeros(2, 4, 64), torch.zeros(4, 16, 2, 64), _i32(1, 2), _i32(1), _i32(2),
                                torch.zeros(1, 2, 32))


def _call(scale=0.125, bs=16, observe=0, decay=1.0, ws=None, nbytes=0, **change):
    b16 = torch.bfloat16
    a = dict(q=torch.zeros(5, 8, 64, dtype=b16), k=torch.zeros(10, 16, 2, 64, dtype=b16), tables=_i32(2, 3), lens=_i32(2),
             start=_i32(3), ks=None, w=torch.zeros(2, 2, 48))
    a.update(change)
    d = {n: None if t is None else _abi.descriptor(t) for n, t in a.items()}
    for x in d.values():
        if x is not None:
            x.t.device = _abi.SFA_ROCM  # reach the checks; every call here is refused before a launch
    r = [_abi.ref(d[n]) for n in ("q", "k", "tables", "lens", "start", "ks")]
    return _abi.lib().cf_chunk_weights(*r, scale, bs, observe, _abi.ref(d["w"]), decay, ws, nbytes, None)


F8 = torch.zeros(10, 16, 2, 64, dtype=torch.float8_e4m3fn)


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(5, 8, 64)), "q: dtype"),
    (dict(q=torch.zeros(5, 7, 64, dtype=torch.bfloat16)), "multiple of num_kv_heads"),
    (dict(q=torch.zeros(5, 8, 128, dtype=torch.bfloat16)), "head_dim"),
    (dict(k=torch.zeros(10, 16, 2, 64)), "k_cache: dtype"),
    (dict(k=torch.zeros(10, 8, 2, 64, dtype=torch.bfloat16)), "block dim"),
    (dict(bs=8), "block_size must be 16"),
    (dict(k=F8), "need k_scale"),
    (dict(ks=torch.ones(2)), "f8e4m3fn caches only"),
    (dict(k=F8, ks=torch.ones(3)), "k_scale: expected 2 or 1"),
    (dict(start=_i32(2)), "q_start must have 3"),
    (dict(start=torch.zeros(3, dtype=torch.int64)), "q_start: expected i32"),
    (dict(lens=_i32(3)), "seq_lens has 3"),
    (dict(tables=torch.zeros(2, 3, dtype=torch.int64)), "block_tables: expected i32"),
    (dict(w=torch.zeros(2, 8, 48)), "one account a KV head, or one for all"),
    (dict(w=torch.zeros(2, 2, 47)), "weights has 47 slots"),
    (dict(w=torch.zeros(2, 1, 48).expand(2, 2, 48)), "rows overlap"),
    (dict(scale=float("inf")), "finite"),
    (dict(decay=float("nan")), "finite"),
    (dict(observe=-1), "observe"),
])
def test_refusals(change, message):
    assert _call(**change) == _abi.CF_ERR_INVALID
    assert message in _abi.last_error()


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(10, 16, 2, 64, dtype=torch.float16)),
    dict(q=torch.zeros(5, 8, 96, dtype=torch.bfloat16), k=torch.zeros(10, 16, 2, 96, dtype=torch.bfloat16)),
    dict(q=torch.zeros(5, 130, 64, dtype=torch.bfloat16)),
    dict(k=torch.zeros(10, 16, 64, 2, dtype=torch.bfloat16).transpose(2, 3)),
    dict(q=torch.zeros(5, 8, 68, dtype=torch.bfloat16)[..., :64]),
])
def test_what_is_not_supported(change):
    assert _call(**change) == _abi.CF_ERR_UNSUPPORTED
    assert "chunk weights" in _abi.last_error()


def test_the_workspace_is_checked():
    need = 1 << 40
    assert _call() == _abi.CF_ERR_WORKSPACE
    assert _call(ws=264, nbytes=need) == _abi.CF_ERR_INVALID and "aligned" in _abi.last_error()
    with pytest.raises(ValueError, match="block_size"):
        ops.chunk_weights_workspace_bytes(5, 2, 8, 2, 64, 3, 8)
    with pytest.raises(ValueError, match="64 query heads"):
        ops.chunk_weights_workspace_bytes(5, 2, 130, 2, 64, 3)
    # 8 bytes a row, head and run of its tokens, 4 a token and head for each run
    # of columns, 4 a row and 4 a block of 256 tokens
    small = ops.chunk_weights_workspace_bytes(5, 2, 8, 2, 64, 3)
    assert 5 * 8 * 8 + 2 * 2 * 48 * 4 <= small <= 4096
    long = ops.chunk_weights_workspace_bytes(8192, 1, 32, 8, 128, 8192)
    assert long <= 64 * 8192 * 32 * 8 + (8192 * 4 // 256 + 1) * 8 * 8192 * 16 * 4 + 512
    # a window of observers needs its rows only
    few = ops.chunk_weights_workspace_bytes(8192, 1, 32, 8, 128, 8192, observe=64)
    assert few <= 33 * 64 * 32 * 8 + 5 * 8 * 8192 * 16 * 4 + 64 * 4 + 512 * 4 + 1024


def test_attention_over_its_own_queries_leaves_none_for_the_accounts():
    slabs = [{"slab_id": n, "storage": "paged", "dims": {"layers": 1, "heads": 2, "dim": 64}, "layout": "BNLD",
              "dtype": "bfloat16"} for n in "kv"]
    mgr = CacheManager({"slabs": slabs, "intercepts": [], "block_size": 16}, num_blocks=4, device="cpu")
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    args = (q, 0, _i32(1, 2), _i32(1), _i32(2))
    with pytest.raises(ValueError, match="out must not be q"):
        mgr.attend_chunks(*args, weights=torch.zeros(1, 2, 32), out=q)
    with pytest.raises(ValueError, match="ROCm"):  # (without accounts the call goes on to the kernels)
        mgr.attend_chunks(*args, out=q)
