"""linear_cross_entropy at the ends of its sizes."""
from __future__ import annotations

import pytest
import torch

from test_gpu_loss import inputs, step

pytestmark = pytest.mark.gpu


def test_no_rows_and_a_weight_past_4_gib(gpu):
    from fused3s_amd.torch_ops import linear_cross_entropy
    V, K = 8_400_001, 512
    w = torch.ones(V, K, dtype=torch.bfloat16, device="cuda").requires_grad_()
    x = torch.zeros(0, K, dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    spare = torch.full((V, K), float("nan"), dtype=torch.bfloat16, device="cuda")
    del spare   # (what the gradient's memory may hold before)
    g, = torch.autograd.grad(linear_cross_entropy(x, w, t, reduction="sum"), [w])
    assert g.shape == (V, K) and not g.any()


@pytest.mark.parametrize("size", [1e-33, 1e-36, 1e-38])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K,V", [(64, 47), (64, 500), (264, 500)])
def test_gradients_near_the_least(gpu, K, V, dtype, size):
    """The loss's gradient near float32's least, all of it or but for one row: those of the
    inputs are what the formula leaves of it, 0 in binary16."""
    x, w, b, t, dloss = inputs(300, K, V, dtype, 6, reduction="none")
    for one in (False, True):
        g = dloss.sign() * size
        if one:
            g[7] = 1.0
            t[7] = 3
        got = step(x, w, b, t, g, "none")
        for name, v in got.items():
            assert bool(torch.isfinite(v).all()), name
        few = step(x[7:8], w, b, t[7:8], g[7:8], "none")
        rest = torch.arange(300, device="cuda") != 7
        # (a row's is at most twice its gradient times the largest weight)
        most = 2 * size * float(w.double().abs().max())
        least = 2.0 ** -24 if dtype == torch.float16 else 0.0
        assert bool((got["dx"][rest].double().abs() <= most * 1.01 + least).all())
        if one:
            # (the logits' gradient, 2 in all, and the result rounded by eps / 2 on either side)
            off = (got["dx"][7].double() - few["dx"][0].double()).abs()
            eps = torch.finfo(dtype).eps
            assert bool((off <= eps * (few["dx"][0].double().abs() + most / size)).all())
