"""torch_ops.linear, activation(x W^T + b) + residual and its gradient, against
64 bits: every value within the type's rounding and the bound of its 32-bit sums."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
F = torch.nn.functional
ACTS = {None: lambda z: z, "relu": F.relu, "gelu": F.gelu, "silu": F.silu,
        "gelu_tanh": lambda z: F.gelu(z, approximate="tanh")}
# What is left of an activation's value and slope beside its rounding to float32:
# Phi to 2e-7 and z Phi to 6e-7, hardware exponentials and reciprocals to a few
# units of float32's last place, for |z| up to 2^6 in the exponent.
ACT_ABS = 2.0 ** -17
STEP = 2.0 ** -24


def make(n, K, M, dtype, bias=True, residual=True, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + n + 7 * K + 31 * M)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    return {"x": rand(n, K).to(dtype), "w": (rand(M, K) * K ** -0.5).to(dtype),
            "b": rand(M).to(dtype) if bias else None,
            "r": rand(n, M).to(dtype) if residual else None, "dy": rand(n, M).to(dtype)}


def step(t, act, leaves="xwbr"):
    from fused3s_amd.torch_ops import linear
    a = {k: v.detach().clone().requires_grad_(k in leaves) if v is not None else None
         for k, v in t.items() if k != "dy"}
    y = linear(a["x"], a["w"], a["b"], act, a["r"])
    names = [k for k in "xwbr" if a[k] is not None and k in leaves]
    grads = torch.autograd.grad(y, [a[k] for k in names], t["dy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}


def check(t, act, got):
    dtype = t["x"].dtype
    half = torch.finfo(dtype).eps / 2
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    x, w, dy = (t[k].double() for k in ("x", "w", "dy"))
    b = t["b"].double() if t["b"] is not None else torch.zeros(w.shape[0], device="cuda").double()
    r = t["r"].double() if t["r"] is not None else torch.zeros_like(dy)
    n, K = x.shape
    M = w.shape[0]
    z = (x @ w.t() + b).requires_grad_()
    a = ACTS[act](z)
    (slope,) = torch.autograd.grad(a.sum(), z)
    z, a = z.detach(), a.detach()
    # z: K + 2 half-steps of the sum of sizes; |act'|, |act''| <= 1.2 (relu: its
    # slope is one of two values where z is that near 0)
    ez = (K + 2) * STEP * (x.abs() @ w.abs().t() + b.abs())
    approx = 0.0 if act in (None, "relu") else ACT_ABS
    ey = 1.2 * ez + approx * (1 + z.abs()) + 2 * STEP * (a.abs() + r.abs())
    if act is None:
        es = torch.zeros_like(z)
    elif act == "relu":
        es = (z.abs() <= ez).double()
    else:
        es = 1.2 * ez + approx * (1 + z.abs()) ** 2
    dz = dy * slope
    # dz is rounded to the type for the products; its columns' sums are not
    edz = dy.abs() * es * (1 + half)
    rdz = edz + (dz.abs() + edz) * half + least if act else edz
    out = {
        "y": (a + r, ey),
        "dx": (dz @ w, rdz @ w.abs() + (M + 2) * STEP * (dz.abs() @ w.abs())),
        "dw": (dz.t() @ x, rdz.t() @ x.abs() + (n + 2) * STEP * (dz.abs().t() @ x.abs())),
        "db": (dz.sum(0), edz.sum(0) + (n + 2) * STEP * dz.abs().sum(0)),
        "dr": (dy, torch.zeros_like(dy)),
    }
    for name, v in got.items():
        want, bound = out[name]
        bound = bound * (1 + half) + want.abs() * half + least
        err = (v.double() - want).abs()
        assert v.dtype == dtype and bool(torch.isfinite(v).all()), name
        worst = float((err / bound).max()) if err.numel() else 0.0
        assert worst <= 1.0, f"{name}: {worst:.3g} times its bound"


SIZES = [
    (1, 8, 8), (1, 1024, 520), (2, 7, 3), (16, 64, 17), (17, 100, 33), (33, 1024, 128),   # few rows
    (64, 40, 300), (65, 8, 8), (65, 9, 5), (100, 72, 136), (127, 65, 129), (128, 64, 64),
    (300, 2048, 65), (300, 2056, 72),                                      # split contraction
    (1003, 100, 301), (1000, 128, 384), (2000, 333, 64), (515, 512, 1032),
    (4100, 264, 1096), (16400, 72, 512), (33000, 16, 136),                  # 128 x 128 tiles
    (49_152, 8, 32), (49_167, 64, 96), (50_001, 136, 416), (49_153, 256, 224),   # W in LDS
    (60_000, 128, 640),
]


@pytest.mark.parametrize("n,K,M", SIZES)
def test_sizes(gpu, n, K, M):
    for i, dtype in enumerate(HALF):
        act = [None, "relu", "gelu", "gelu_tanh", "silu"][(n + K + i) % 5]
        t = make(n, K, M, dtype, bias=(n + M) % 3 > 0, residual=(K + M + i) % 2 > 0)
        check(t, act, step(t, act))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("n,K,M", [(5, 48, 40), (400, 96, 160), (20000, 32, 264)])
def test_activations(gpu, n, K, M, act, dtype):
    t = make(n, K, M, dtype, seed=3)
    check(t, act, step(t, act))
    t["b"] = t["b"] * 8          # far into both tails
    check(t, act, step(t, act))


def test_some_gradients(gpu):
    """Any subset of the inputs may ask for gradients; they are what all get."""
    t = make(500, 64, 72, torch.float16)
    for act in (None, "gelu"):
        every = step(t, act)
        for leaves in ("x", "w", "b", "r", "xb", "wr"):
            for name, g in step(t, act, leaves).items():
                assert torch.equal(g, every[name]), (leaves, name)


@pytest.mark.parametrize("n,K,M", [
    (404, 45, 4037), (66, 4104, 520), (500, 4096, 72),       # deep dx, deep z: split
    (3000, 512, 517), (9000, 1024, 1030), (70, 8, 8200),     # operands whole, outputs odd
    (2500, 2048, 2056), (300, 1027, 1025)])
def test_products_of_a_step(gpu, n, K, M):
    """Every way a step's products take through tiles, with and without the sums
    that a bias needs."""
    for i, dtype in enumerate(HALF):
        for act, bias in ((None, bool(i)), ("silu" if i else "gelu", True)):
            t = make(n, K, M, dtype, bias=bias, residual=bias, seed=4)
            check(t, act, step(t, act))


@pytest.mark.parametrize("dtype", HALF)
def test_many_rows_gradients(gpu, dtype):
    """Rows enough for W in LDS, in both passes: blocks of rows that do not divide
    among the workgroups, outputs that need two turns of 384, a last row alone, no
    bias, a bias but no gradient of it; every run gives the same bits."""
    for n, K, M, act, bias in ((49_169, 128, 416, "gelu", True), (70_001, 64, 800, "silu", True),
                               (49_152, 248, 224, "gelu_tanh", True),
                               (98_304, 416, 136, None, True), (98_321, 32, 256, "relu", True),
                               (50_000, 32, 32, "relu", False)):
        t = make(n, K, M, dtype, bias=bias, residual=False, seed=2)
        got = step(t, act)
        check(t, act, got)
        for name, g in step(t, act, "xw").items():
            assert torch.equal(g, got[name]), (n, name)


@pytest.mark.parametrize("act", [None, "silu"])
def test_layouts(gpu, act):
    """Rows at a distance, unaligned starts, transposed weights, more dimensions,
    expanded gradients: the bits of contiguous inputs in the same kernels, within
    the bound in others."""
    from fused3s_amd.torch_ops import linear
    t = make(200, 64, 72, torch.float16, seed=5)
    want = step(t, act)
    wide = torch.zeros(200, 200, dtype=torch.float16, device="cuda")
    wide[:, 8:72] = t["x"]
    res = torch.zeros(200, 88, dtype=torch.float16, device="cuda")
    res[:, 16:] = t["r"]
    wt = t["w"].t().contiguous().t()
    assert not wt.is_contiguous()
    y = linear(wide[:, 8:72], wt, t["b"], act, res[:, 16:])
    assert torch.equal(y, want["y"])
    odd = torch.zeros(200, 73, dtype=torch.float16, device="cuda")
    odd[:, 1:65] = t["x"]
    got = {**t, "x": odd[:, 1:65]}
    a = odd[:, 1:65].detach().requires_grad_()
    y = linear(a, t["w"], t["b"], act, t["r"])
    (dx,) = torch.autograd.grad(y, a, t["dy"])
    check(got, act, {"y": y.detach(), "dx": dx})
    x3 = t["x"].view(5, 40, 64)
    y = linear(x3, t["w"], t["b"], act, t["r"].view(5, 40, 72))
    assert y.shape == (5, 40, 72) and torch.equal(y.view(200, 72), want["y"])
    one = linear(t["x"][3], t["w"], t["b"], act, t["r"][3])
    assert one.shape == (72,)
    check({k: (v[3:4] if k in "xr" or k == "dy" else v) for k, v in t.items()}, act,
          {"y": one[None]})
    a = t["x"].clone().requires_grad_()
    row = t["r"][:1].clone().requires_grad_()
    linear(a, t["w"], t["b"], act, row.expand(200, 72)).sum().backward()
    ones = {**t, "r": row.detach().expand(200, 72).contiguous(), "dy": torch.ones_like(t["dy"])}
    assert torch.equal(a.grad, step(ones, act)["dx"])
    assert torch.equal(row.grad, torch.full_like(row, 200.0))


def test_no_rows(gpu):
    t = make(0, 64, 72, torch.float16)
    for act in (None, "gelu"):
        got = step(t, act)
        assert got["y"].shape == (0, 72) and got["dx"].shape == (0, 64)
        assert not got["dw"].any() and not got["db"].any()


def test_odd_values(gpu):
    """An infinite or NaN input reaches its own row only, and infinite weights
    their own output; past the last row nothing is written."""
    from fused3s_amd.torch_ops import linear
    for n in (10, 300):
        t = make(n, 100, 64, torch.float16)
        clean = linear(t["x"], t["w"], t["b"], "gelu", t["r"])
        x = t["x"].clone()
        x[4, 99] = float("nan")
        y = linear(x, t["w"], t["b"], "gelu", t["r"])
        rest = torch.arange(n, device="cuda") != 4
        assert torch.equal(y[rest], clean[rest]) and torch.isnan(y[4]).all()
        w = t["w"].clone()
        w[63, 0] = float("inf")
        y = linear(t["x"], w, t["b"], None, t["r"])
        assert torch.isfinite(y[:, :63]).all() and not torch.isfinite(y[:, 63]).any()


def test_relu_of_nan_is_nan(gpu):
    from fused3s_amd.torch_ops import linear
    x = torch.full((3, 8), float("nan"), dtype=torch.bfloat16, device="cuda")
    w = torch.ones(8, 8, dtype=torch.bfloat16, device="cuda")
    assert torch.isnan(linear(x, w, activation="relu")).all()


def test_large_rows(gpu):
    """Row offsets past 2^31 and 2^32 bytes, in both directions."""
    from fused3s_amd.torch_ops import linear
    n, K, M = 1_100_000, 2048, 16
    x = torch.zeros(n, K, dtype=torch.float16, device="cuda")
    assert x.numel() * 2 > 2**32
    rows = torch.tensor([0, 1, 524_287, 524_288, 1_048_575, 1_048_576, n - 1], device="cuda")
    t = make(7, K, M, torch.float16, residual=False)
    x[rows] = t["x"]
    dy = torch.zeros(n, M, dtype=torch.float16, device="cuda")
    dy[rows] = t["dy"]
    x.requires_grad_()
    w = t["w"].clone().requires_grad_()
    y = linear(x, w, t["b"], "relu")
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    check(t, "relu", {"y": y.detach()[rows], "dx": dx[rows], "dw": dw})
    assert torch.equal(y.detach()[5], torch.relu(t["b"]))


def test_deterministic_streams_capture(gpu):
    """The same bits on any stream, in parallel, and from a replayed graph with
    eager work in between."""
    t = make(700, 1032, 200, torch.float16)
    want = step(t, "gelu")
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(step(t, "gelu"))
    torch.cuda.synchronize()
    for other in got:
        for name in want:
            assert torch.equal(other[name], want[name]), name
    static = {k: v.clone() for k, v in t.items()}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(static, "gelu")
    for seed in range(3):
        fresh = make(700, 1032, 200, torch.float16, seed=seed)
        for k in static:
            static[k].copy_(fresh[k])
        g.replay()
        torch.cuda.synchronize()
        eager = step(fresh, "gelu")
        for name in eager:
            assert torch.equal(out[name], eager[name]), (seed, name)


def test_refusals(gpu):
    from fused3s_amd.torch_ops import linear
    t = make(20, 16, 24, torch.float16)
    x, w, b, r = (t[k] for k in "xwbr")
    for args in ((x.float(), w), (x.cpu(), w), (x, w.bfloat16()), (x, w, b.float()),
                 (x[:, :8], w), (x, w[0]), (x, w, b[:8]), (x, w, b, "tanh"),
                 (x, w, b, None, r[:5]), (x, w, b, None, r[:1]), (x[:, :0], w[:, :0])):
        with pytest.raises(ValueError):
            linear(*args)
    leaf = x.clone().requires_grad_()
    (d,) = torch.autograd.grad(linear(leaf, w, b, "silu").sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), leaf)
