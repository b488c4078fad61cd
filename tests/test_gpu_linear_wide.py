"""linear() at sizes that take its large tiles: many tiles per workgroup, ends
inside tiles, the errors' size and the same bits from run to run."""
from __future__ import annotations

import pytest
import torch

from _linear_sizes import WIDE
from test_gpu_linear_act import HALF, check, make, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", HALF)
def test_roundings_of_a_step(gpu, dtype):
    """y and db are rounded once.  dz is rounded to the type before dx and dw are
    made of it: that rounding passes through a product with the relative size it
    has, independent of the result's own, so together they are sqrt(2) of one.  (Of
    8 M values: 2 % above what rounding the 64-bit result leaves.)"""
    t = make(8200, 1024, 1032, dtype, residual=False, seed=6)
    got = step(t, "gelu")
    check(t, "gelu", got)
    leaves = [t[k].double().requires_grad_() for k in "xwb"]
    z = leaves[0] @ leaves[1].t() + leaves[2]
    y = torch.nn.functional.gelu(z)
    want = {"y": y.detach(), **dict(zip(("dx", "dw", "db"),
                                        torch.autograd.grad(y, leaves, t["dy"].double())))}
    for name, times in (("y", 1.0), ("db", 1.0), ("dx", 2 ** 0.5), ("dw", 2 ** 0.5)):
        one = (want[name].to(dtype).double() - want[name]).norm()
        slack = 1.02 if name != "db" else 1.25   # (1,032 values)
        assert (got[name].double() - want[name]).norm() <= times * slack * one, name
    for _ in range(3):
        for name, v in step(t, "gelu").items():
            assert torch.equal(v, got[name]), name


@pytest.mark.parametrize("n,K,M", WIDE)
def test_wide(gpu, n, K, M):
    """Every product of a step, both types, with an activation (a slope pass, dW alone)
    and without (db beside dW), every epilogue; each value within its bound."""
    acts = ["relu", "gelu", "gelu_tanh", "silu"]
    for i, dtype in enumerate(HALF):
        for act, bias, residual in ((acts[(n + K + 2 * i) % 4], True, i == 0), (None, i == 1, i == 1)):
            t = make(n, K, M, dtype, bias=bias, residual=residual, seed=9)
            got = step(t, act)
            check(t, act, got)
            again = step(t, act, "xw")
            for name, v in again.items():
                assert torch.equal(v, got[name]), (name, act)
            del t, got, again


def test_wide_rows_without_a_gradient_are_kept(gpu):
    """dy of 0 in all rows but some, which lie in the last tiles of a workgroup: the
    others' dx is 0, dW and db are those rows' alone."""
    n, K, M = 12_300, 1000, 4104
    t = make(n, K, M, torch.bfloat16, residual=False, seed=10)
    rows = torch.tensor([0, 255, 256, 8191, 8192, 12_287, 12_288, 12_299], device="cuda")
    dy = torch.zeros_like(t["dy"])
    dy[rows] = t["dy"][rows]
    got = step({**t, "dy": dy}, "gelu")
    small = {**{k: t[k][rows] for k in ("x", "dy")}, "w": t["w"], "b": t["b"], "r": None}
    check(small, "gelu", {"dx": got["dx"][rows], "dw": got["dw"], "db": got["db"]})
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert not got["dx"][rest].any()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n", [3, 300, 49_170])
def test_gelu_tails(gpu, n, dtype):
    """gelu, its derivative and the other activations over z from -12 to 12: z Phi(z) to
    6e-7 absolute (its fit), and what 16 bits leave.  K = 8 inputs give z exactly: one
    is z, the others 0."""
    import math
    from test_gpu_linear_act import ACTS
    M, half = 64, torch.finfo(dtype).eps / 2
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    # y[i][m] = act(x[i] . w[m]): x[i] = row i's start, w[m] = 1, and bias 0: so a row
    # has one z; the bias spreads it, both of few bits
    x = torch.zeros(n, 8, device="cuda", dtype=dtype)
    x[:, 0] = (torch.arange(n, device="cuda") % 24 - 12).to(dtype)
    w = torch.zeros(M, 8, device="cuda", dtype=dtype)
    w[:, 0] = 1.0
    b = (torch.arange(M, device="cuda") / 64.0).to(dtype)
    z = x[:, :1].double() + b.double()
    t = {"x": x, "w": w, "b": b, "r": None,
         "dy": torch.ones(n, M, device="cuda", dtype=dtype)}
    for act in ("gelu", "gelu_tanh", "silu"):
        got = step(t, act)
        zz = z.clone().requires_grad_()
        want = ACTS[act](zz)
        (slope,) = torch.autograd.grad(want.sum(), zz)
        # values: 6e-7 (gelu's fit; the others' exponential and reciprocal, a few
        # 2^-24 of |z| <= 12, are less), then one rounding
        err = (got["y"].double() - want).abs()
        assert bool((err <= (6e-7 + want.abs() * half + least) * (1 + 2.0 ** -7)).all()), act
        # db: n slopes of 2e-7 + 12 x 2^-22 each, summed in float32
        err = (got["db"].double() - slope.sum(0)).abs()
        bound = n * (2e-7 + 12 * 2.0 ** -22) + (n + 2) * 2.0 ** -24 * slope.abs().sum(0)
        assert bool((err <= bound + slope.sum(0).abs() * half + least).all()), act
        assert math.isfinite(float(got["dx"].double().sum()))
