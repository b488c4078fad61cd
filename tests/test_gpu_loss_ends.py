"""linear_cross_entropy at the ends of its sizes."""
from __future__ import annotations

import pytest
import torch

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
