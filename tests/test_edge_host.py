"""Edge attention's host side on any host: what the C entry points refuse before they
touch a device, and the 64-bit reference's gradient against differences."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import _edge_reference as reference
from conftest import random_csr
from fused3s_amd import _lib


def test_entry_points_refuse():
    h = _lib.hip()
    need = C.c_int64()
    assert h.f3s_edge_attention_workspace(None, None, 0, C.byref(need)) == 1
    call = lambda plan=None, n=16, dtype=0, cap=0.0, pos=None, dims=0, slopes=None: \
        h.f3s_edge_attention_fwd(plan, 16, 64, 16, 64, 16, 64, 16, 64, None, dtype, n, 1, 1.0, cap,
                                 pos, dims, slopes, None, 0, None)
    assert call() == 1                 # no plan
    assert b"plan" in h.f3s_last_error()
    assert call(n=-1) == 1 and call(dtype=2) == 1
    for cap in (-1.0, float("nan"), float("inf"), 1e-35):
        assert call(cap=cap) == 1 and b"cap" in h.f3s_last_error()
    for bad in (dict(dims=4, pos=16, slopes=16), dict(dims=-1), dict(dims=1, pos=16),
                dict(dims=1, slopes=16)):
        assert call(**bad) == 1 and b"positions" in h.f3s_last_error()
    assert h.f3s_edge_attention_bwd(None, None, 16, 64, 16, 64, 16, 64, 16, 16, 64, 16, 64, 16, 64,
                                    16, 64, None, 0, 16, 1, 1.0, 0.0, None, 0, None, None, 0,
                                    None) == 1


@pytest.mark.parametrize("cap,dims", [(None, 0), (2.0, 0), (None, 1), (3.0, 3)])
def test_reference_gradient(cap, dims):
    """The formula's gradient is the derivative of the formula: differences of the
    64-bit forward pass, step 2^-13 (third derivatives of size 1 leave 2^-28)."""
    n, H, scale = 9, 2, 0.3
    rp, ci = random_csr(n, 3, 5, self_loops=False)
    gen = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen)
    q, k, v, do = (rand(n, H, 64).half() for _ in range(4))
    positions = rand(n, dims) if dims else None
    slopes = rand(H) if dims else None
    ref = reference.Reference(q, k, v, do, rp, ci, scale, cap, positions, slopes)
    adj = reference.adjacency(n, rp, ci)
    x = {"q": q.double(), "k": k.double(), "v": v.double()}
    if dims:
        x["slopes"] = slopes.double()
    at = lambda **changed: reference.forward(
        **{"slopes": None, **x, **changed}, positions=positions, adj=adj, scale=scale, cap=cap)
    assert torch.allclose(at(), ref.value["o"])
    step = 2.0 ** -13
    for name in x:
        d = torch.randn(x[name].shape, generator=gen, dtype=torch.float64)
        got = (ref.value["d" + name].view_as(d) * d).sum()
        want = (do.double() * (at(**{name: x[name] + step * d})
                               - at(**{name: x[name] - step * d}))).sum() / (2 * step)
        size = (ref.value["d" + name].view_as(d).abs() * d.abs()).sum()
        assert abs(got - want) <= 2.0 ** -15 * size, name
