"""f3s_linear_fwd / _bwd write nothing behind the workspace they asked for or behind
their results, whichever gradients are wanted."""
from __future__ import annotations

import ctypes as C
import itertools

import pytest
import torch

from test_gpu_linear_act import check, make

pytestmark = pytest.mark.gpu

GUARD = 4096


def guarded(nbytes):
    """`nbytes` of device memory and a guard behind them."""
    t = torch.full((nbytes + GUARD,), 0xa5, dtype=torch.uint8, device="cuda")
    return t, lambda: bool((t[nbytes:] == 0xa5).all())


def workspace(n, K, M, act, backward):
    from fused3s_amd import _lib
    need = C.c_int64()
    assert _lib.hip().f3s_linear_workspace(n, K, M, act, backward, C.byref(need)) == 0
    return need.value


@pytest.mark.parametrize("n,K,M", [
    (70, 8, 8), (300, 2048, 65), (404, 45, 4037), (1000, 128, 384), (2500, 2048, 2056),
    (300, 1027, 1025), (700, 1032, 1032), (512, 1024, 2048), (4096, 2048, 2048), (1100, 4, 2048),
    (49_170, 64, 96)])
@pytest.mark.parametrize("act", [0, 1])
def test_bounds(gpu, n, K, M, act):
    from fused3s_amd import _lib
    h, stream = _lib.hip(), torch.cuda.current_stream().cuda_stream
    t = make(n, K, M, torch.float16, residual=False, seed=8)
    name = ("none", "relu")[act]
    size = workspace(n, K, M, act, 0)
    ws, kept = guarded(size)
    y, y_kept = guarded(2 * n * M)
    assert h.f3s_linear_fwd(t["x"].data_ptr(), K, t["w"].data_ptr(), t["b"].data_ptr(), None, 0,
                            y.data_ptr(), n, K, M, act, 0, ws.data_ptr(), size, stream) == 0
    assert kept() and y_kept()
    check(t, None if act == 0 else name, {"y": y[:2 * n * M].view(torch.float16).view(n, M)})
    size = workspace(n, K, M, act, 1)
    shapes = {"dx": (n, K), "dw": (M, K), "db": (M,)}
    for wanted in itertools.product((0, 1), repeat=3):
        ws, kept = guarded(size)
        out = {k: guarded(2 * s.numel()) for k, s in
               ((k, torch.empty(s, device="meta")) for k, s in shapes.items())}
        ptrs = [out[k][0].data_ptr() if w else None for k, w in zip(shapes, wanted)]
        assert h.f3s_linear_bwd(t["x"].data_ptr(), K, t["w"].data_ptr(), t["b"].data_ptr(),
                                t["dy"].data_ptr(), M, *ptrs, n, K, M, act, 0, ws.data_ptr(),
                                size, stream) == 0
        assert kept() and all(g() for _, g in out.values()), wanted
        got = {k: out[k][0][:-GUARD].view(torch.float16).view(shapes[k])
               for k, w in zip(shapes, wanted) if w}
        check(t, None if act == 0 else name, got)
