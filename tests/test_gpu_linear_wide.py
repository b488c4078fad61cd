"""linear() at sizes that take its large tiles: many tiles per workgroup, ends
inside tiles, the errors' size and the same bits from run to run."""
from __future__ import annotations

import pytest
import torch

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
