"""Edge attention with nodes infinitely far: they are taken out of the graph, forward and
backward, edges between two of them included."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _edge_reference import Reference
from conftest import random_csr
from test_gpu_edge import inputs, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap,dims", [(None, 1), (3.0, 2), (None, 3)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,H", [(250, 1), (4000, 5)])
def test_nodes_infinitely_far(gpu, n, H, dtype, cap, dims):
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(n, 5, 4)   # (with loops)
    x = inputs(n, H, dtype, 3, dims)
    x["slopes"] = x["slopes"].abs() + 0.1
    far = np.zeros(n, bool)
    far[::7] = True
    rows = np.repeat(np.arange(n), np.diff(rp))
    assert (far[rows] & far[ci] & (rows != ci)).any()
    positions = x["positions"].view(n, dims).clone()
    at = torch.as_tensor(np.flatnonzero(far)).cuda()
    sign = torch.where(torch.arange(at.numel(), device="cuda") % 3 == 0, -1.0, 1.0)
    positions[at, torch.arange(at.numel(), device="cuda") % dims] = sign * float("inf")
    got = step(TorchGraph(rp, ci, heads=H), {**x, "positions": positions.view_as(x["positions"])}, cap=cap)
    keep = ~far[ci] & ~far[rows]
    rp2 = np.concatenate([[0], np.cumsum(np.bincount(rows[keep], minlength=n))]).astype(np.int32)
    ref = Reference(x["q"], x["k"], x["v"], x["do"], rp2, ci[keep], 0.125, cap, x["positions"],
                    x["slopes"])
    for name, t in got.items():
        ref.check(name, t)
        if name != "dslopes":
            assert not t[at].any(), name
