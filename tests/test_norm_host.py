"""Layer norm's host side on any host: what the C entry points and the binding refuse
before they touch a device, and the 64-bit reference's gradient against differences."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import _norm_reference as reference
from fused3s_amd import _lib


def test_entry_points_refuse():
    h = _lib.hip()
    need = C.c_int64()
    size = lambda n, width, dtype=0: h.f3s_layer_norm_workspace(n, width, dtype, C.byref(need))
    assert size(-1, 8) == 1 and size(1, 0) == 1 and size(1, 8, 3) == 1
    assert size(1, 1 << 24) == 5 and size(1 << 40, 8) == 5
    assert h.f3s_layer_norm_workspace(4, 8, 0, None) == 1
    assert size(0, 8) == 0 and need.value == 0
    assert size(5, 8) == 0 and need.value >= 2 * 8 * 4
    fwd = lambda x=16, stride=8, y=16, stats=None, n=4, width=8, dtype=0, wtype=0: \
        h.f3s_layer_norm_fwd(x, stride, None, None, y, stats, n, width, 1e-5, dtype, wtype, None)
    assert fwd(x=None) == 1 and fwd(y=None) == 1 and fwd(stride=7) == 1 and fwd(stats=4) == 1
    assert fwd(dtype=0, wtype=1) == 1      # neither x's type nor float32
    assert fwd(n=-1) == 1 and fwd(width=1 << 24, stride=1 << 24) == 5
    assert fwd(n=0) == 0                   # nothing to do
    bwd = lambda stats=16, dy=8, ws=16, size=1 << 20, dw=16: h.f3s_layer_norm_bwd(
        16, 8, None, stats, 16, dy, 16, dw, None, 4, 8, 0, 0, ws, size, None)
    assert bwd(stats=None) == 1 and bwd(dy=4) == 1 and bwd(ws=None) == 1 and bwd(size=8) == 1
    assert b"workspace" in h.f3s_last_error()


def test_workspace_grows_with_the_rows_up_to_the_resident_ones():
    h = _lib.hip()
    need = C.c_int64()
    for dtype in (0, 1, 2):
        for width in (1, 8, 301, 1024, 5000, 16384, 100_000):
            last = 0
            for n in (1, 17, 4096, 1 << 22, 1 << 30):
                assert h.f3s_layer_norm_workspace(n, width, dtype, C.byref(need)) == 0
                assert need.value >= last
                last = need.value
            assert last <= 1024 * 2 * width * 4


def test_binding_refuses():
    from fused3s_amd.torch_ops import layer_norm
    x = torch.zeros(4, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        layer_norm(x)
    with pytest.raises(ValueError, match="weight must have shape"):
        layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="bias must have shape"):
        layer_norm(x, None, torch.ones(1, 8))
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(torch.zeros(()))


def test_reference_gradient():
    """The formula's gradient is the derivative of the formula, and both are torch's."""
    gen = torch.Generator().manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).float()
    x, w, b, dy = rand(5, 11), rand(11), rand(11), rand(5, 11)
    ref = reference.Reference(x, w, b, dy, 1e-3)
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (11,), leaves[1], leaves[2], 1e-3)
    assert torch.allclose(y, ref.value["y"], rtol=1e-12, atol=1e-12)
    for name, g in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy.double())):
        assert torch.allclose(g, ref.value[name], rtol=1e-11, atol=1e-11), name
    step = 2.0 ** -13
    for i, name in enumerate(("dx", "dw", "db")):
        d = torch.randn(leaves[i].shape, generator=gen, dtype=torch.float64)
        value = []
        for s in (step, -step):
            a = [t.detach() + (s * d if j == i else 0) for j, t in enumerate(leaves)]
            c = a[0] - a[0].mean(1, keepdim=True)
            h = c * ((c * c).mean(1, keepdim=True) + 1e-3) ** -0.5
            value.append(((h * a[1] + a[2]) * dy.double()).sum())
        got = (ref.value[name] * d).sum()
        assert abs(got - (value[0] - value[1]) / (2 * step)) <= 2.0 ** -16 * \
            (ref.value[name].abs() * d.abs()).sum(), name
