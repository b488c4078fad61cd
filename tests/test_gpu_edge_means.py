"""The gradient of edge attention's queries where the values have a large mean: every edge of
a row has nearly the same do.v, and dq is made of the differences."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _edge_reference import adjacency, scores, softmax
from conftest import random_csr
from test_gpu_edge import hub_csr, step

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("cap,dims", [(None, 0), (4.0, 2)])
@pytest.mark.parametrize("mean", [16, 64])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,H,hubs", [(300, 2, False), (5601, 3, True), (9000, 2, False)])
def test_values_of_a_large_mean(gpu, n, H, hubs, dtype, mean, cap, dims):
    """Whole numbers, so that every product and do.v is exact: dq within what the differences
    of do.v from their mean leave, and as near as the columns' gradients."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = hub_csr(n, 5, 3) if hubs else random_csr(n, 12, 3)
    gen = torch.Generator(device="cuda").manual_seed(n + mean)
    whole = lambda low, high: torch.randint(low, high + 1, (n, H, 64), generator=gen,
                                            device="cuda").to(dtype)
    x = {"q": whole(-1, 1), "k": whole(-1, 1), "v": whole(mean - 3, mean + 3), "do": whole(0, 2)}
    if dims:
        x["positions"] = torch.rand(n, dims, generator=gen, device="cuda")
        x["slopes"] = 0.5 + 0.5 * torch.rand(H, generator=gen, device="cuda")
    got = step(TorchGraph(rp, ci, heads=H), x, cap=cap)
    adj = adjacency(n, rp, ci).cuda()
    rows = lambda a: a.double().transpose(0, 1).contiguous()
    cols = lambda a: a.transpose(-1, -2).contiguous()
    Q, K, V, dO = (rows(x[name]) for name in ("q", "k", "v", "do"))
    s, c, dist = scores(*(x[name].double() for name in ("q", "k")), x.get("positions"),
                        x.get("slopes"), 0.125, cap)
    p = softmax(s, adj)
    g = torch.matmul(dO, cols(V))
    away = g - (p * g).sum(-1, keepdim=True)
    # weights are within 2^-17 of themselves as two values of bfloat16, 2^-22 of binary16 (and
    # of a row's largest); exponents and c by the roundings of scores below 2^6
    f16 = dtype == torch.float16
    e = (2.0 ** -22 if f16 else 2.0 ** -17) + 2.0 ** -16 + 64 * 2.0 ** -22
    # what is taken from do.v is one of the row's, as far from their mean as the farthest: in
    # p (do.v - it), in p times the mean's distance from it, and twice in that mean
    far = away.masked_fill(~adj, 0.0).abs().amax(-1, keepdim=True)
    size = p * (away.abs() + 4 * far)
    # do.v's mean is a float32 sum and quotient of float32 products, and the difference from
    # it is rounded: four half-steps of do.v's size (a row of one edge has away = far = 0, and
    # its dq is what these leave)
    rest = p * 2.0 ** -22 * g.abs().masked_fill(~adj, 0.0).amax(-1, keepdim=True)
    half, least = torch.finfo(dtype).eps / 2, 2.0 ** -25 if f16 else 2.0 ** -134
    out = lambda a: a.transpose(0, 1)
    exact = out(torch.matmul(p * away * c, K)) * 0.125
    floor = (2.0 ** -22 * size.amax(-1, keepdim=True)) * adj
    bound = out(torch.matmul(e * size + rest + floor, K.abs())) * 0.125
    bound = bound * (1 + half) + half * exact.abs() * (1 + 2.0 ** -10) + least
    err = (got["dq"].double() - exact).abs()
    assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} times its bound"
    if dims:
        want = -(p * away * dist).sum((1, 2))
        # (a row's sums are of some 2^13 edges at most, added in chains of 2^9 and less)
        err = (got["dslopes"].double() - want).abs()
        assert bool((err <= (((e + 2.0 ** -15) * size + rest) * dist).sum((1, 2)) + 2.0 ** -24 * want.abs()).all())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n", [120, 17_000])
def test_a_weight_near_the_least(gpu, n, dtype):
    """Rows whose do.v are all the same but for that of one edge, whose weight is 2^-80 to
    2^-140: dq is finite and what that edge leaves of it, within the columns' bound."""
    from _edge_reference import Reference
    from fused3s_amd.torch_ops import TorchGraph
    rows, width = 48, 100   # (rows of `width` edges; the others have a loop each)
    rp = np.concatenate([np.arange(rows + 1) * width,
                         rows * width + np.arange(1, n - rows + 1)]).astype(np.int32)
    ci = np.concatenate([np.tile(np.arange(width), rows), np.arange(rows, n)]).astype(np.int32)
    x = {name: torch.zeros(n, 1, 64, device="cuda") for name in ("q", "k", "v", "do")}
    for name, value in (("v", 1.0), ("do", 1.0)):
        x[name][:] = value
    low = 60                               # the one edge's other end, in a later chunk
    x["v"][low] = 3.0
    x["q"][:rows, 0, 0] = torch.linspace(55, 97, rows, device="cuda").floor()
    x["k"][low, 0, 0] = -1.0
    x["k"][:width, 0, 1] = 1.0
    x = {name: t.to(dtype) for name, t in x.items()}
    got = step(TorchGraph(rp, ci, heads=1), x, scale=1.0)
    few = slice(0, 100)                    # (all edges of these rows are among these nodes)
    small = {name: t[few] for name, t in x.items()}
    rp = np.concatenate([rp[:rows + 1], rp[rows] + np.arange(1, 100 - rows + 1)]).astype(np.int32)
    ref = Reference(*(small[name] for name in ("q", "k", "v", "do")), rp, ci[:rp[-1]], 1.0)
    for name in ("o", "dq", "dk", "dv"):
        ref.check(name, got[name][few])
