"""linear_cross_entropy's host side on any host: what the C entry points and the binding
refuse before they touch a device, workspaces, and the 64-bit reference against torch's
own loss and against differences."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import _loss_reference as reference
from fused3s_amd import _lib


def test_entry_points_refuse():
    h = _lib.hip()
    need = C.c_int64()
    size = lambda n, K, V, back=0: h.f3s_cross_entropy_workspace(n, K, V, back, C.byref(need))
    assert size(-1, 8, 8) == 1 and size(1, 0, 8) == 1 and size(1, 8, 0) == 1
    assert size(1, 1 << 22, 8) == 5 and size(1, 8, 1 << 30) == 5 and size(1 << 31, 8, 8) == 5
    assert h.f3s_cross_entropy_workspace(1, 8, 8, 0, None) == 1
    assert size(0, 8, 8) == 0 and need.value == 0
    fwd = lambda x=16, stride=8, w=16, target=16, loss=16, n=4, how=1, dtype=0, ws=16, size=1 << 20: \
        h.f3s_cross_entropy_fwd(x, stride, w, None, target, -100, loss, None, n, 8, 8, how, dtype,
                                ws, size, None)
    for bad in (dict(x=8), dict(w=8), dict(stride=12), dict(stride=1 << 22),   # (16-byte rows)
                dict(x=None), dict(w=None), dict(target=None), dict(loss=None), dict(stride=7),
                dict(n=-1), dict(how=3), dict(how=-1), dict(dtype=2), dict(ws=None), dict(ws=8),
                dict(size=8)):
        assert fwd(**bad) == 1, bad
    bwd = lambda lse=16, dloss=16, ws=16, size=1 << 30: h.f3s_cross_entropy_bwd(
        16, 8, 16, None, 16, -100, lse, dloss, 16, 16, None, 4, 8, 8, 1, 0, ws, size, None)
    assert h.f3s_cross_entropy_bwd(16, 8, 16, None, 16, -100, 16, 16, 16, 24, None, 4, 8, 8, 1, 0,
                                   16, 1 << 30, None) == 1   # (dW at 8 bytes past a 16)
    assert bwd(lse=None) == 1 and bwd(dloss=None) == 1 and bwd(ws=None) == 1 and bwd(size=8) == 1
    assert b"workspace" in h.f3s_last_error()


def test_workspace_goes_with_a_piece_of_the_classes():
    """Not with n V: the backward pass's for a million classes is a piece's.  (Fewer
    classes may need more: what few inputs leave goes with the shares of the classes.)"""
    h = _lib.hip()
    need = C.c_int64()
    for K in (64, 264):
        for back in (0, 1):
            for V in (2, 47, 1000, 50_021, 1_000_000):
                assert h.f3s_cross_entropy_workspace(16_384, K, V, back, C.byref(need)) == 0
                # (logits in 16 bits of a million: 33 GB)
                assert 0 < need.value < 2**30, (K, V, back)


def test_workspace_of_padded_copies():
    """Rows of K inputs that are no whole pieces: with many rows and classes, copies of rows
    that are, beside what those take."""
    h = _lib.hip()
    need = C.c_int64()
    def size(n, K, back):
        assert h.f3s_cross_entropy_workspace(n, K, 10_000, back, C.byref(need)) == 0
        return need.value
    for n, K, Kp, copied in ((999, 41, 41, False), (1000, 41, 48, True), (5000, 257, 264, True),
                             (5000, 48, 48, False)):
        for back in (0, 1):
            copies = (1 + back) * 2 * Kp * (n + 10_000) if copied else 0
            assert 0 <= size(n, K, back) - size(n, Kp, back) - copies < 1024 or not copied


def test_binding_refuses():
    from fused3s_amd.torch_ops import linear_cross_entropy
    x, w = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(5, 8, dtype=torch.float16)
    t = torch.zeros(4, dtype=torch.int64)
    for args, what in (((x, w, t), "GPU"), ((x, w[:, :7], t), "do not fit"),
                       ((x, w[:0], t), "empty"), ((x, w, t[:3]), "target must have shape"),
                       ((x, w, t, torch.zeros(4)), "bias must have shape"),
                       ((x, w, t, None, -100, "max"), "reduction")):
        with pytest.raises(ValueError, match=what):
            linear_cross_entropy(*args)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reference(reduction):
    gen = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=gen)
    x, w, b = rand(7, 5).half(), rand(11, 5).half(), rand(11).half()
    t = torch.tensor([0, 10, -100, 3, 3, 7, -100])
    dloss = rand(7) if reduction == "none" else rand(())
    ref = reference.Reference(x, w, b, t, reduction, dloss)
    leaves = [v.double().requires_grad_() for v in (x, w, b)]
    loss = torch.nn.functional.cross_entropy(torch.nn.functional.linear(*leaves), t,
                                             reduction=reduction)
    assert torch.allclose(loss, ref.value["loss"], rtol=1e-12)
    for name, g in zip(("dx", "dw", "db"), torch.autograd.grad(loss, leaves, dloss.double())):
        assert torch.allclose(g, ref.value[name], rtol=1e-11, atol=1e-13), name
    step = 2.0 ** -13
    for i, name in enumerate(("dx", "dw", "db")):
        d = torch.randn(leaves[i].shape, generator=gen, dtype=torch.float64)
        value = []
        for s in (step, -step):
            a = [v.detach() + (s * d if j == i else 0) for j, v in enumerate(leaves)]
            z = a[0] @ a[1].t() + a[2]
            each = (torch.logsumexp(z, 1) - z.gather(1, t.clamp(min=0)[:, None])[:, 0]) * (t != -100)
            each = each / (5 if reduction == "mean" else 1)
            value.append((each * dloss.double()).sum())
        got = (ref.value[name] * d).sum()
        size = (ref.value[name].abs() * d.abs()).sum()
        assert abs(got - (value[0] - value[1]) / (2 * step)) <= 2.0 ** -16 * size, name
