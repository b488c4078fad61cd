"""linear()'s gradients of no rows, beside a weight of more than 2^32 values."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_rows_and_a_weight_past_4_gib(gpu):
    from fused3s_amd.torch_ops import linear
    M, K = 4_100_001, 1056
    w = torch.ones(M, K, dtype=torch.bfloat16, device="cuda").requires_grad_()
    x = torch.zeros(0, K, dtype=torch.bfloat16, device="cuda")
    spare = torch.full((M, K), float("nan"), dtype=torch.bfloat16, device="cuda")
    del spare   # (what the gradient's memory may hold before)
    y = linear(x, w)
    g, = torch.autograd.grad(y, [w], torch.zeros_like(y))
    assert g.shape == (M, K) and not g.any()
