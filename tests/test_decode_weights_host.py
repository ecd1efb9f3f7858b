"""Decode with accounts without a GPU: refusals and the workspace."""

from __future__ import annotations

import ctypes

import pytest
import torch

from cf_hip import _abi, ops
from kernels.paged_attention import paged_attention_weights


def test_cpu_tensors_are_refused():
    q, k = torch.zeros(1, 4, 64), torch.zeros(4, 16, 2, 64)
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm"):
        paged_attention_weights(q, k, k, t, n, torch.zeros(1, 2, 32))


def _call(decay=1.0, ws=None, nbytes=0, bs=16, **change):
    a = dict(q=torch.zeros(2, 8, 64), k=torch.zeros(10, 16, 2, 64), v=torch.zeros(10, 16, 2, 64),
             tables=torch.zeros(2, 3, dtype=torch.int32), lens=torch.zeros(2, dtype=torch.int32), shared=None, ks=None,
             vs=None, w=torch.zeros(2, 2, 48), out=torch.zeros(2, 8, 64))
    a.update(change)
    d = {n: None if t is None else _abi.descriptor(t) for n, t in a.items()}
    for x in d.values():
        if x is not None:
            x.t.device = _abi.SFA_ROCM  # reach the checks; every call here is refused before a launch
    r = [_abi.ref(d[n]) for n in ("q", "k", "v", "tables", "lens", "shared", "ks", "vs")]
    return _abi.lib().cf_paged_decode_weights(*r, 0.125, bs, _abi.ref(d["w"]), decay, _abi.ref(d["out"]), ws, nbytes,
                                              None)


@pytest.mark.parametrize("change, message", [
    (dict(w=None), "weights"),
    (dict(w=torch.zeros(2, 2, 48, dtype=torch.float64).to(torch.float16)), "weights: expected f32"),
    (dict(w=torch.zeros(2, 4, 48)), "one account a KV head, or one for all"),
    (dict(w=torch.zeros(3, 2, 48)), "weights must be"),
    (dict(w=torch.zeros(2, 2, 47)), "weights has 47 slots"),
    (dict(w=torch.zeros(2, 2, 96)[:, :, ::2]), "the last stride must be 1"),
    (dict(w=torch.zeros(1, 2, 48).expand(2, 2, 48)), "rows overlap"),
    (dict(decay=float("inf")), "decay"),
    (dict(bs=0), "block_size"),
    (dict(bs=8), "block dim"),
    (dict(out=torch.zeros(2, 8, 32)), "out shape"),
    (dict(shared=torch.zeros(3, dtype=torch.int32)), "shared_prefix_lens has 3"),
    (dict(ks=torch.ones(2)), "f8e4m3fn caches only"),
])
def test_refusals(change, message):
    assert _call(**change) == _abi.CF_ERR_INVALID
    assert message in _abi.last_error()


def test_the_workspace_is_checked():
    assert _call() == _abi.CF_ERR_WORKSPACE
    need = ops.decode_weights_workspace_bytes(2, 8, 2, 64, 3, 16)
    assert _call(ws=256, nbytes=need - 1) == _abi.CF_ERR_WORKSPACE and str(need) in _abi.last_error()
    assert _call(ws=264, nbytes=need) == _abi.CF_ERR_INVALID and "aligned" in _abi.last_error()


def test_the_workspace_holds_a_score_a_head_and_token():
    n, plain = ctypes.c_uint64(), ctypes.c_uint64()
    lib = _abi.lib()
    for b, hq, h, d, mb, bs in ((64, 32, 8, 128, 512, 16), (1, 12, 12, 64, 1, 16), (3, 6, 2, 40, 7, 8), (0, 4, 4, 64, 3, 16)):
        assert lib.cf_paged_decode_weights_workspace_bytes(b, hq, h, d, mb, bs, ctypes.byref(n)) == 0
        assert lib.cf_paged_decode_workspace_bytes(b, hq, h, d, mb, bs, 512, ctypes.byref(plain)) == 0
        row = (mb * bs + 31) // 32 * 32
        assert plain.value + b * hq * (row * 4 + 8) <= n.value <= plain.value + b * hq * (row * 4 + 8) + 512
    assert lib.cf_paged_decode_weights_workspace_bytes(1, 5, 2, 64, 3, 16, ctypes.byref(n)) == _abi.CF_ERR_INVALID
    assert lib.cf_paged_decode_weights_workspace_bytes(1, 4, 2, 64, 3, 0, ctypes.byref(n)) == _abi.CF_ERR_INVALID
    assert lib.cf_paged_decode_weights_workspace_bytes(1, 4, 2, 64, 3, 1000, ctypes.byref(n)) == 0


def test_the_workspace_query_refuses_a_null_result():
    assert _abi.lib().cf_paged_decode_weights_workspace_bytes(1, 4, 2, 64, 3, 16, None) == _abi.CF_ERR_INVALID
    assert "bytes_out is NULL" in _abi.last_error()
