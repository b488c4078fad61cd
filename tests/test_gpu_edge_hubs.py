"""Edge attention of a row with one large weight and tens of thousands of small, equal ones:
the small ones' sum keeps its precision."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [3000, 60_000])
def test_many_small_weights(gpu, n, dtype, first):
    from fused3s_amd.torch_ops import TorchGraph
    hubs = 48
    rp = np.concatenate([np.arange(hubs + 1) * n, hubs * n + np.arange(1, n - hubs + 1)]).astype(np.int32)
    ci = np.concatenate([np.tile(np.arange(n), hubs), np.arange(hubs, n)]).astype(np.int32)
    heavy = 1 if first else n - 1
    # hub i's score is (10 + i / 16) for the heavy node, 0 for the others; values of 1, the
    # heavy one's 0
    q, k, v = (torch.zeros(n, 1, 64, device="cuda") for _ in range(3))
    score = 10 + torch.arange(hubs, device="cuda").double() / 16   # (exact in 8 bits)
    score = score.to(dtype).double()
    q[:hubs, 0, 0], k[heavy, 0, 0] = score.float(), 1.0
    v[:] = 1.0
    v[heavy] = 0.0
    graph = TorchGraph(rp, ci, heads=1)
    got = graph.edge_attention(*(t.to(dtype) for t in (q, k, v)), 1.0)[:hubs, 0].double()
    want = ((n - 1) / (n - 1 + torch.exp(score)))[:, None].expand(hubs, 64)
    half = torch.finfo(dtype).eps / 2
    # A weight as two 16-bit values is within 2^-22 (binary16) or 2^-17 of itself, and its
    # exponent within 2^-20; n of them in chains of n / 32 adds of float32 (their sum and the
    # weights' own); binary16's end 2^-31 below a row's largest.
    e = (2.0 ** -22 if dtype == torch.float16 else 2.0 ** -17) + 2.0 ** -19 + n / 32 * 2.0 ** -24
    floor = 2.0 ** -31 * n if dtype == torch.float16 else 0.0
    largest = torch.exp(score)[:, None] / (n - 1 + torch.exp(score))[:, None]
    bound = half * want * (1 + 2.0 ** -10) + e * want + floor * largest
    err = (got - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
