"""layer_norm and its gradient against 64 bits: every value within the type's rounding
and the bound of its 32-bit sums."""
from __future__ import annotations

import pytest
import torch

from _norm_reference import Reference

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]
# lanes of a wave, of one or two pieces, workgroups of one and two pieces, rows read in
# turns; whole pieces, ragged ends and rows below a piece
SHAPES = [(1, 1), (1, 2), (3, 7), (2, 8), (5, 9), (33, 31), (7, 64), (70, 100), (33, 128), (65, 129),
          (16, 255), (9, 301), (17, 512), (5, 513), (3, 1000), (3, 1024), (3, 1025), (4, 2047),
          (3, 4096), (2, 4097), (3, 8192), (2, 8193), (2, 16384), (2, 16385), (3, 40_001),
          (4099, 40), (20_011, 8), (1, 100_000)]


def inputs(n, C, dtype, of, seed, shift=0.3, scale=1.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    return ((rand(n, C) * scale + shift).to(dtype), (1 + 0.3 * rand(C)).to(of),
            (0.3 * rand(C)).to(of), rand(n, C).to(dtype))


def step(x, w, b, dy, eps=1e-5):
    from fused3s_amd.torch_ops import layer_norm
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, eps=eps)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    names = ["dx"] + (["dw"] if w is not None else []) + (["db"] if b is not None else [])
    return {"y": y.detach(), **dict(zip(names, grads))}


def check(got, x, w, b, dy, eps=1e-5):
    ref = Reference(x, w, b, dy, eps)
    for name, t in got.items():
        ref.check(name, t)


@pytest.mark.parametrize("wide", [False, True], ids=["same", "float32"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,C", SHAPES)
def test_step(gpu, n, C, dtype, wide):
    from fused3s_amd.torch_ops import layer_norm
    x = inputs(n, C, dtype, torch.float32 if wide else dtype, n + C)
    got = step(*x)
    check(got, *x)
    with torch.no_grad():
        assert torch.equal(layer_norm(*x[:3]), got["y"])
    again = step(*x)
    for name in got:
        assert torch.equal(got[name], again[name]), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [5, 128, 301, 1024, 2900, 40_000])
@pytest.mark.parametrize("has", [(0, 0), (1, 0), (0, 1)])
def test_without_weights(gpu, C, dtype, has):
    x, w, b, dy = inputs(6, C, dtype, dtype, C)
    x = (x, w if has[0] else None, b if has[1] else None, dy)
    check(step(*x), *x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [7, 64, 301, 2050, 20_000])
def test_rows_apart_and_unaligned(gpu, C, dtype):
    """Slices of wider matrices, from any column on; a weight of the same kind; gradients
    that are broadcast or transposed."""
    from fused3s_amd.torch_ops import layer_norm
    wide, w, b, dy = inputs(9, C + 5, dtype, dtype, C)
    x, w, b = wide[:, 3:3 + C], w[1:1 + C], b[2:2 + C]
    dys = [dy[:, 1:1 + C], dy[:, :C].t().contiguous().t(), dy[:1, :C].expand(9, C),
           dy[:, :1].expand(9, C)]
    for g in dys:
        check(step(x, w, b, g), x, w, b, g)
    leaf = x.detach().requires_grad_()
    layer_norm(leaf, w, b).sum().backward()
    ref = Reference(x, w, b, torch.ones(9, C, device="cuda"), 1e-5)
    ref.check("dx", leaf.grad)


@pytest.mark.parametrize("dtype", TYPES)
def test_shapes(gpu, dtype):
    from fused3s_amd.torch_ops import layer_norm
    x, w, b, _ = inputs(24, 32, dtype, dtype, 3)
    y = layer_norm(x, w, b)
    assert torch.equal(layer_norm(x.view(2, 3, 4, 32), w, b), y.view(2, 3, 4, 32))
    assert torch.equal(layer_norm(x[0], w, b), y[0])
    assert torch.equal(layer_norm(x.view(4, 6, 32).transpose(0, 1), w, b),
                       y.view(4, 6, 32).transpose(0, 1))
    leaves = [t.detach().requires_grad_() for t in (x[:0], w, b)]
    out = layer_norm(*leaves)
    assert out.shape == (0, 32) and out.dtype is dtype
    for g, leaf in zip(torch.autograd.grad(out, leaves, torch.zeros_like(out)), leaves):
        assert g.shape == leaf.shape and not g.any()
    leaves = [x.view(2, 12, 32).detach().requires_grad_(), w, b.detach().requires_grad_()]
    g = torch.autograd.grad(layer_norm(*leaves).sum(), [leaves[0], leaves[2]])
    assert g[0].shape == (2, 12, 32) and torch.equal(g[1], torch.full_like(b, 24))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [64, 300, 5000])
def test_hard_rows(gpu, C, dtype):
    """Means far above the spread, rows of one value, tiny and large values."""
    shift = {torch.float16: 100.0, torch.bfloat16: 16.0, torch.float32: 1000.0}[dtype]
    x, w, b, dy = inputs(8, C, dtype, dtype, C, shift=shift, scale=1.0)
    x[1] = 3.0
    x[2] = 0.0
    x[3] = (x[3].float() * 1e-3).to(dtype)
    x[4] = (x[4].float() * (300.0 if dtype is torch.float16 else 1e8)).clamp(-6e4, 6e4).to(dtype) \
        if dtype is torch.float16 else (x[4].float() * 1e8).to(dtype)
    check(step(x, w, b, dy, eps=1e-3), x, w, b, dy, eps=1e-3)


def test_odd_values_stay_in_their_row(gpu):
    """Infinite and NaN values reach their own row and, in the weights' gradients, what
    is summed over it."""
    for C in (64, 301, 5000, 40_000):
        x, w, b, dy = inputs(40, C, torch.bfloat16, torch.float32, 1)
        clean = step(x, w, b, dy)
        x[17, 5], x[39, 0] = float("nan"), float("inf")
        got = step(x, w, b, dy)
        rest = [i for i in range(40) if i not in (17, 39)]
        for name in ("y", "dx"):
            assert torch.equal(got[name][rest], clean[name][rest]), name
            assert got[name][[17, 39]].isnan().all(), name
        assert got["dw"].isnan().all() and torch.equal(got["db"], clean["db"])


@pytest.mark.parametrize("n,C", [(17_000_001, 128), (40_000, 56_000)])
def test_past_32_bit_offsets(gpu, n, C):
    """Rows at both ends and between; the others' dy is 0."""
    _, w, b, dy = inputs(90, C, torch.bfloat16, torch.bfloat16, 13)
    x = torch.randn(n, C, device="cuda", dtype=torch.bfloat16)
    some = torch.cat([torch.arange(30), n // 2 + torch.arange(30), n - 30 + torch.arange(30)]).cuda()
    whole = torch.zeros(n, C, device="cuda", dtype=torch.bfloat16)
    whole[some] = dy
    got = step(x, w, b, whole)
    for name in ("y", "dx"):
        got[name] = got[name][some]
    check(got, x[some], w, b, dy)


def test_other_stream_and_capture(gpu):
    """On a stream of its own, and captured and replayed with new inputs, each replay
    against the eager result."""
    from fused3s_amd.torch_ops import layer_norm
    x, w, b, dy = inputs(1000, 256, torch.bfloat16, torch.float32, 5)
    want = step(x, w, b, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(s)
    for name in want:
        assert torch.equal(got[name], want[name]), name
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    with torch.cuda.stream(s):
        torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(*leaves)
        grads = torch.autograd.grad(y, leaves, dy)
    for seed in range(3):
        new = inputs(1000, 256, torch.bfloat16, torch.float32, 50 + seed)
        with torch.no_grad():
            for t, value in zip((*leaves, dy), new):
                t.copy_(value)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*new)
        for name, t in zip(("y", "dx", "dw", "db"), (y, *grads)):
            assert torch.equal(t, want[name]), name


def test_refusals(gpu):
    from fused3s_amd.torch_ops import layer_norm
    x, w, b, _ = inputs(4, 8, torch.float16, torch.float16, 1)
    with pytest.raises(ValueError):
        layer_norm(x.double())
    with pytest.raises(ValueError):
        layer_norm(x, w.bfloat16())
    with pytest.raises(ValueError):
        layer_norm(x, w, b.float())
    with pytest.raises(ValueError):
        layer_norm(x, w.cpu())
    with pytest.raises(ValueError):
        layer_norm(x, None, b.bfloat16())
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        layer_norm(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="traced"):
        torch.func.vmap(layer_norm)(x)
