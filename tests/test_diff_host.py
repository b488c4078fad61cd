"""Differential attention's host side on any host: what the C entry points
refuse before they touch a device, and the 64-bit reference's gradient against
differences."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import _diff_reference as reference
from conftest import random_csr
from fused3s_amd import _lib


def test_entry_points_refuse():
    h = _lib.hip()
    need = C.c_int64()
    assert h.f3s_diff_attention_workspace(None, None, C.byref(need)) == 1
    call = lambda plan=None, n=16, H=1, dtype=0: h.f3s_diff_attention_fwd(
        plan, 16, 128, 16, 128, 16, 128, 16, 16, 128, None, dtype, n, H, 1.0, None, 0, None)
    assert call() == 1                 # no plan
    assert b"plan" in h.f3s_last_error()
    assert call(n=-1) == 1
    assert call(dtype=2) == 1
    assert h.f3s_diff_attention_bwd(None, None, 16, 128, 16, 128, 16, 128, 16, 16, 16, 128, 16, 128,
                                    16, 128, 16, 128, 16, 0, 16, 1, 1.0, None, 0, None) == 1
    assert h.f3s_reverse_csr(None, None, 4, 0, None, None, None) == 1
    assert h.f3s_reverse_csr(16, 16, 0, 4, 16, 16, None) == 1
    assert h.f3s_reverse_csr(16, 16, -1, 0, 16, 16, None) == 1
    p = C.c_void_p()
    assert h.f3s_plan_create_scheduled(None, 4, 1, None, C.byref(p)) == 1
    assert h.f3s_plan_create_scheduled(16, 4, 65, None, C.byref(p)) == 1


def test_scheduled_plan_takes_no_order():
    from fused3s_amd import Plan

    class Bsf:
        window_offsets = W = None

    with pytest.raises(ValueError, match="scheduled"):
        Plan(Bsf(), seg_tiles=4, scheduled=True)


def test_reference_gradient():
    """The formula's gradient is the derivative of the formula: differences of the
    64-bit forward pass, step 2^-13 (third derivatives of size 1 leave 2^-28)."""
    n, H, scale = 9, 2, 0.3
    rp, ci = random_csr(n, 3, 5, self_loops=False)
    gen = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen).half()
    q, k, v, do = (rand(n, H, 128) for _ in range(4))
    lam = torch.tensor([0.4, 1.3])
    ref = reference.Reference(q, k, v, lam, do, rp, ci, scale)
    adj = reference.adjacency(n, rp, ci)
    x = {"q": q.double(), "k": k.double(), "v": v.double(), "lam": lam.double()}

    def loss(**changed):
        return (do.double() * reference.forward(**{**x, **changed}, adj=adj, scale=scale)).sum()

    assert torch.allclose(reference.forward(**x, adj=adj, scale=scale), ref.value["o"])
    step = 2.0 ** -13
    for name in x:
        d = torch.randn(x[name].shape, generator=gen, dtype=torch.float64)
        got = (ref.value["d" + name].view_as(d) * d).sum()
        want = (loss(**{name: x[name] + step * d}) - loss(**{name: x[name] - step * d})) / (2 * step)
        size = (ref.value["d" + name].view_as(d).abs() * d.abs()).sum()
        assert abs(got - want) <= 2.0 ** -15 * size, name
