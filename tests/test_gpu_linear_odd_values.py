"""linear()'s gradient where z or dy are infinite, NaN or at the type's ends, in
each kernel that a backward pass takes."""
from __future__ import annotations

import pytest
import torch

from test_gpu_linear_act import ACTS, HALF, make, step

pytestmark = pytest.mark.gpu

# the slope's kernel: split z and its join, whole tiles, tiles with operands through
# registers, W in LDS
SIZES = [(70, 4104, 72), (400, 96, 160), (401, 97, 161), (49_170, 64, 96)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,K,M", SIZES)
def test_relu_passes_on_or_not(gpu, n, K, M, dtype):
    """An off unit's gradient is 0 whatever dy is; an on unit's is dy, infinite or
    not, and reaches its own row of dx and its own output's dw and db."""
    t = make(n, K, M, dtype, residual=False, seed=1)
    t["b"][0], t["b"][1], t["b"][8] = -1000.0, 1000.0, -1000.0   # off, on, off in every row
    clean = step(t, "relu")
    for value in (float("inf"), float("nan")):
        bad = {**t, "dy": t["dy"].clone()}
        bad["dy"][3, 0] = bad["dy"][n - 1, 8] = value
        assert torch.equal(bad["x"], t["x"])
        got = step(bad, "relu")
        for name in got:
            assert torch.equal(got[name], clean[name]), (name, value)
        bad["dy"][5, 1] = value
        got = step(bad, "relu")
        rows = torch.arange(n, device="cuda") != 5
        outs = torch.arange(M, device="cuda") != 1
        assert torch.equal(got["dx"][rows], clean["dx"][rows])
        assert torch.equal(got["dw"][outs], clean["dw"][outs])
        assert torch.equal(got["db"][outs], clean["db"][outs])
        assert not torch.isfinite(got["dx"][5]).any() and not torch.isfinite(got["db"][1])


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("n,K,M", SIZES)
def test_odd_rows_stay_alone(gpu, n, K, M, act):
    """A NaN or infinite value in one row of x or dy: the other rows of dx are bit
    for bit what they are without it."""
    t = make(n, K, M, torch.float16, residual=False, seed=2)
    clean = step(t, act)
    rows = torch.arange(n, device="cuda") != 7
    for name in ("x", "dy"):
        for value in (float("inf"), float("nan")):
            bad = {**t, name: t[name].clone()}
            bad[name][7, 3] = value
            got = step(bad, act)
            assert torch.equal(got["dx"][rows], clean["dx"][rows]), (name, value)
            assert torch.equal(got["y"][rows], clean["y"][rows]), (name, value)
            if name == "dy":
                outs = torch.arange(M, device="cuda") != 3
                assert torch.equal(got["dw"][outs], clean["dw"][outs]), value
                assert torch.equal(got["db"][outs], clean["db"][outs]), value


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("n,K,M", SIZES)
def test_gradient_of_large_products(gpu, n, K, M, act):
    """z of any finite size (bfloat16 reaches 2^127): the slope is 0 or 1, not what an
    overflow on the way makes of it."""
    t = make(n, K, M, torch.bfloat16, residual=False, seed=3)
    t["w"] = t["w"] * 2.0 ** -60          # (the columns below are their bias)
    exps = [10, 20, 40, 63, 64, 65, 90, 120]
    for i, e in enumerate(exps):
        t["b"][2 * i], t["b"][2 * i + 1] = 2.0 ** e, -2.0 ** e
    got = step(t, act)
    on, off = slice(0, 2 * len(exps), 2), slice(1, 2 * len(exps), 2)
    assert torch.isfinite(got["y"]).all()
    assert torch.equal(got["y"][:, on], t["b"][on].expand(n, -1)) and not got["y"][:, off].any()
    # db: n values of dy summed in float32, rounded once
    dy = t["dy"][:, on].double()
    bound = (n + 2) * 2.0 ** -24 * dy.abs().sum(0) + 2.0 ** -8 * dy.sum(0).abs()
    assert ((got["db"][on].double() - dy.sum(0)).abs() <= bound).all()
    assert not got["db"][off].any()
    assert all(torch.isfinite(g).all() for g in got.values())


def test_one_row_of_any_stride(gpu):
    """A single row's stride means nothing, however large or odd."""
    from fused3s_amd.torch_ops import TorchGraph, linear
    import numpy as np
    t = make(1, 64, 72, torch.float16)
    want = step(t, "silu")
    graph = TorchGraph(np.array([0, 1], np.int32), np.zeros(1, np.int32), heads=1)
    row = torch.randn(1, 3 * 128, device="cuda").half()
    lam = torch.tensor([0.5], device="cuda")
    o = graph.diff_attention_packed(row, lam, 0.125)
    for stride in (0, 1, 7, 2 ** 22, 2 ** 30, 2 ** 31 + 1):
        x, r = (t[k].as_strided(t[k].shape, (stride, 1)) for k in "xr")
        assert torch.equal(linear(x, t["w"], t["b"], "silu", r), want["y"]), stride
        odd = row.as_strided(row.shape, (stride, 1))
        leaf = odd.detach().requires_grad_()
        again = graph.diff_attention_packed(leaf, lam, 0.125)
        assert torch.equal(again, o), stride
        again.sum().backward()
        q, k, v = (odd[:, 128 * i:128 * i + 128] for i in range(3))
        assert torch.equal(graph.diff_attention(q, k, v, lam, 0.125), o), stride
        q = q.view(1, 1, 128).as_strided((1, 1, 128), (stride, 3, 1))
        assert torch.equal(graph.diff_attention(q, k, v, lam, 0.125), o), stride
