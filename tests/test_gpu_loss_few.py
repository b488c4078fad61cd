"""The gradients of the loss of few classes: the logits' gradient is not rounded to the type
on its way to those of x and weight."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_loss import inputs, step

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,K,V,reduction", [(1, 8, 2, "none"), (300, 64, 7, "none"), (1003, 128, 47, "mean"),
                                             (20_011, 128, 47, "mean"), (2000, 72, 64, "none"),
                                             (515, 256, 33, "none"), (3000, 200, 16, "mean"),
                                             (129, 32, 17, "sum"), (40_000, 48, 3, "mean")])
def test_one_rounding(gpu, n, K, V, reduction, dtype):
    x, w, b, t, dloss = inputs(n, K, V, dtype, n + K + V, reduction=reduction)
    got = step(x, w, b, t, dloss, reduction)
    counted = t != -100
    div = max(int(counted.sum()), 1) if reduction == "mean" else 1
    mm, T = torch.matmul, lambda a: a.t().contiguous()
    X, W = x.double(), w.double()
    z = mm(X, T(W)) + b.double()
    p = torch.softmax(z, 1)
    g = (dloss.double().expand(n) * counted / div)[:, None]
    d = p.clone()
    d.scatter_add_(1, t.clamp(min=0)[:, None], -torch.ones(n, 1, dtype=torch.float64, device="cuda"))
    dz = d * g
    # a probability's error: its logit's (K + 4 half-steps of its products' sizes), the
    # log-sum-exp's and the exponents' roundings
    err = ((K + 4) * U * (mm(X.abs(), T(W.abs())) + b.double().abs())).amax(1)
    err = err + 2.0 ** -22 * (z.abs().amax(1) + math.log(V) + 1)
    edz = (p * (4 * err[:, None] + 64 * U + 2.0 ** -19) + 2 * U * d.abs()) * g.abs()
    # two 16-bit values for each: 2^-17 (bfloat16), 2^-22 (binary16), which end at half of
    # its least value, of what is 2^14 or more times the largest
    f16 = dtype == torch.float16
    half, least = torch.finfo(dtype).eps / 2, 2.0 ** -25 if f16 else 2.0 ** -134
    floor = least * 2.0 ** -14 * 2 * float(g.abs().max()) if f16 else least
    er = edz + (2.0 ** -22 if f16 else 2.0 ** -17) * (dz.abs() + edz) + floor
    for name, exact, size in (
            ("dx", mm(dz, W), mm(er, W.abs()) + (2 * V + 8) * U * mm(dz.abs() + er, W.abs())),
            ("dw", mm(T(dz), X), mm(T(er), X.abs()) + (2 * n + 8) * U * mm(T(dz.abs() + er), X.abs()))):
        bound = size + half * (exact.abs() * (1 + 2.0 ** -10) + size) + least
        off = (got[name].double() - exact).abs()
        assert bool((off <= bound).all()), f"{name}: {float((off / bound).max()):.3g} times its bound"
