"""torch_ops.linear's host side on any host: what the C entry points and the
Python call refuse before they touch a device, and the workspaces they ask for."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from fused3s_amd import _lib


def test_entry_points_refuse():
    h = _lib.hip()
    need = C.c_int64()
    size = lambda *a: h.f3s_linear_workspace(*a, C.byref(need))
    assert size(-1, 8, 8, 0, 0) == 1
    assert size(8, 0, 8, 0, 0) == 1
    assert size(8, 8, 8, 5, 0) == 1
    assert size(8, 1 << 22, 8, 0, 0) == 5
    assert h.f3s_linear_workspace(8, 8, 8, 0, 0, None) == 1
    fwd = lambda n=8, K=8, M=8, act=0, dtype=0, x=16, xs=8, ws=0: h.f3s_linear_fwd(
        x, xs, 16, None, None, 0, 16, n, K, M, act, dtype, None, ws, None)
    assert fwd(dtype=2) == 1 and fwd(act=-1) == 1 and fwd(x=None) == 1 and fwd(xs=4) == 1
    assert fwd(n=0, x=None) == 0                 # nothing to do
    assert size(1000, 4096, 64, 0, 0) == 0 and need.value > 0
    assert fwd(n=1000, K=4096, M=64, xs=4096) == 1
    assert b"workspace" in h.f3s_last_error()
    bwd = lambda n=8, dy=16, dys=8, ws=None, size=0: h.f3s_linear_bwd(
        16, 8, 16, None, dy, dys, 16, 16, 16, n, 8, 8, 0, 0, ws, size, None)
    assert bwd(dy=None) == 1 and bwd(dys=4) == 1 and bwd() == 1


def test_call_refuses():
    from fused3s_amd.torch_ops import linear
    x, w = torch.zeros(4, 8).half(), torch.zeros(6, 8).half()
    with pytest.raises(ValueError, match="on a GPU"):
        linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="do not fit"):
        linear(x, w.t())
    with pytest.raises(ValueError, match="residual"):
        linear(x, w, residual=torch.zeros(6).half())
    with pytest.raises(ValueError, match="empty"):
        linear(x[:, :0], w[:, :0])
