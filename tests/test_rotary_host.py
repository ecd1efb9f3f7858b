"""Rotary positions without a GPU: refusals, and the plain statement."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from cf_hip import _abi, ops
from kernels.rotary import rotary, rotary_cache_write
from oracle import rotary as oracle


def test_cpu_tensors_and_bad_orders_are_refused():
    x, pos, f = torch.zeros(2, 1, 8), torch.zeros(2, dtype=torch.int64), torch.ones(4)
    with pytest.raises(ValueError, match="ROCm"):
        rotary(x, pos, f)
    with pytest.raises(ValueError, match="ROCm"):
        rotary_cache_write(x, x, x, pos, f, pos, x[None], x[None])
    with pytest.raises(ValueError, match="axis_order"):
        ops._rotary_axes(pos, None, "spiral", False)
    with pytest.raises(ValueError, match="2 sections for 1"):
        ops._rotary_axes(pos, (2, 2), "blocks", False)
    with pytest.raises(ValueError, match="at most 4"):
        ops._rotary_axes(torch.zeros(5, 2), (1, 1, 1, 1, 0), "blocks", False)


def _write(**change):
    a = dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64),
             pos=torch.zeros(3, 3, dtype=torch.int32), f=torch.zeros(32), slots=torch.zeros(3, dtype=torch.int64),
             kc=torch.zeros(5, 16, 2, 64), vc=torch.zeros(5, 16, 2, 64), ks=None, vs=None, out=torch.zeros(3, 4, 64),
             sections=(8, 12, 12), axes=3, flags=0, scale=1.0)
    a.update(change)
    d = {n: _abi.descriptor(t) if isinstance(t, torch.Tensor) else None for n, t in a.items()}
    for x in d.values():
        if x is not None:
            x.t.device = _abi.SFA_ROCM  # reach the checks; every call here is refused before a launch
    r = {n: _abi.ref(x) for n, x in d.items()}
    sec = None if a["sections"] is None else (ctypes.c_int32 * len(a["sections"]))(*a["sections"])
    return _abi.lib().cf_rotary_cache_write(r["q"], r["k"], r["v"], r["pos"], r["f"], sec, a["axes"], a["flags"],
                                            a["scale"], r["slots"], r["kc"], r["vc"], r["ks"], r["vs"], r["out"], None)


F8 = torch.zeros(5, 16, 2, 64, dtype=torch.float8_e4m3fn)


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.int32)), "q: dtype"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.float16)), "k_new dtype"),
    (dict(v=torch.zeros(3, 1, 64)), "v_new has 1 heads"),
    (dict(k=torch.zeros(2, 2, 64)), "k_new must be [3"),
    (dict(out=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "q_out dtype"),
    (dict(out=torch.zeros(3, 1, 64).expand(3, 4, 64)), "rows overlap"),
    (dict(pos=torch.zeros(2, 3, dtype=torch.int32)), "expected [3, T]"),
    (dict(pos=torch.zeros(3, 4, dtype=torch.int32)), "positions: 4 rows"),
    (dict(pos=torch.zeros(3, 3)), "positions: expected i32 or i64"),
    (dict(f=torch.zeros(33)), "do not fit head_dim"),
    (dict(f=torch.zeros(32, dtype=torch.float64)), None),
    (dict(sections=None), "sections are needed"),
    (dict(sections=(8, 12, 11)), "sections sum to 31"),
    (dict(sections=(-1, 12, 21)), "must not be negative"),
    (dict(sections=(8, 12, 12), flags=1), "more pairs than its turns"),
    (dict(axes=5), "axes (5)"),
    (dict(flags=4), "unknown flags"),
    (dict(scale=float("nan")), "rotary_scale"),
    (dict(slots=torch.zeros(2, dtype=torch.int64)), "slot_mapping has 2"),
    (dict(slots=torch.zeros(3)), "slot_mapping: expected i32 or i64"),
    (dict(vc=torch.zeros(5, 16, 2, 64, dtype=torch.float16)), "v_cache dtype"),
    (dict(vc=torch.zeros(4, 16, 2, 64)), "v_cache shape"),
    (dict(kc=F8, vc=F8), "need k_scale"),
    (dict(kc=F8, vc=F8, ks=torch.ones(2)), "need v_scale"),
    (dict(kc=F8, vc=F8, ks=torch.ones(3), vs=torch.ones(2)), "k_scale: expected 2 or 1"),
    (dict(ks=torch.ones(2)), "k_scale applies to f8e4m3fn"),
])
def test_cache_write_refuses(change, message):
    if message is None:  # a type without a code has no descriptor
        with pytest.raises(ValueError, match="float64"):
            _write(**change)
        return
    assert _write(**change) == _abi.CF_ERR_INVALID
    assert message in _abi.last_error()


def test_the_plain_statement():
    """A quarter turn swaps a pair; two turns add up; other axes' positions do not matter."""
    x = np.arange(8.0).reshape(1, 1, 8)
    got, _ = oracle.rotate(x, [[1]], [np.pi / 2, 0.0], [2])
    assert np.allclose(got[0, 0], [-2, 1, 0, 3, 4, 5, 6, 7])
    got, _ = oracle.rotate(x, [[1]], [np.pi / 2, 0.0], [2], adjacent=True)
    assert np.allclose(got[0, 0], [-1, 0, 2, 3, 4, 5, 6, 7])
    assert oracle.axis_of_pair(6, (2, 1, 3), "blocks") == [0, 0, 1, 2, 2, 2]
    assert oracle.axis_of_pair(8, (4, 2, 2), "cycled") == [0, 1, 2, 0, 1, 2, 0, 0]
    f, x = [0.3, 0.7], np.random.default_rng(1).normal(size=(2, 1, 4))
    once, _ = oracle.rotate(x, [[5, 5], [9, 1]], f, (1, 1))
    twice, _ = oracle.rotate(oracle.rotate(x, [[2, 1], [4, 0]], f, (1, 1))[0], [[3, 4], [5, 1]], f, (1, 1))
    assert np.allclose(once, twice)
