"""Differential attention's gradient where weights are far below binary16's normal
range: nodes that rows hardly attend, and rows of very many edges."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _diff_reference import Reference
from test_gpu_diff import HALF, check, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("pairs", [40, 3000])
def test_hardly_attended_nodes(gpu, pairs, dtype):
    """Rows of two edges whose logits are 4 to 14 apart (in both maps, or with a lam
    of 0 in one): the other node's only edge has a weight of 2^-6 to 2^-20.  With
    gradients around 2^10 its dv is a normal number of the type, and held to the
    same relative bound as any.  (3,000: a row per wave.)"""
    from fused3s_amd.torch_ops import TorchGraph
    H, n = 2, 3 * pairs
    gen = torch.Generator(device="cuda").manual_seed(pairs)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    rp = np.minimum(np.arange(n + 1) * 2, 2 * pairs).astype(np.int32)
    ci = (pairs + np.arange(2 * pairs)).astype(np.int32)      # row i: two nodes of its own
    graph = TorchGraph(rp, ci, heads=H)
    q, k, v, do = rand(n, H, 128) * 0.1, rand(n, H, 128) * 0.1, rand(n, H, 128), rand(n, H, 128)
    apart = torch.linspace(4.0, 14.0, pairs, device="cuda")
    q[..., 0] = q[..., 64] = 4.0
    for at in (0, 64):
        k[pairs::2, :, at] = 0.0
        k[pairs + 1::2, :, at] = -apart[:, None] / 4.0
    x = [t.to(dtype) for t in (q, k, v)] + [torch.tensor([0.0, 0.5], device="cuda"),
                                            (do * 1024.0).to(dtype)]
    x[3][1] = 0.5
    got = step(graph, *x, 1.0)
    if pairs < 1000:
        check(got, *x, rp, ci, 1.0)
    ref = Pairs(*x, pairs)
    for name in ("dv", "o"):
        ref.check(name, got[name])


class Pairs:
    """The same rows in 64 bits, without a matrix of all pairs of nodes; bounds as
    Reference's: 66 half-steps of float32 in a logit, 2^-20 (2^-17 bfloat16) in a
    weight, the result's rounding."""

    def __init__(self, q, k, v, lam, do, pairs):
        self.dtype = q.dtype
        d = lambda t: t.double()
        q, k, v, do, lam = d(q[:pairs]), d(k[pairs:]), d(v[pairs:]), d(do[:pairs]), d(lam)
        H = q.shape[1]
        k, v = k.view(pairs, 2, H, 128), v.view(pairs, 2, H, 128)
        prod = q[:, None] * k
        s = prod.view(pairs, 2, H, 2, 64).sum(-1)
        size = float(prod.abs().view(pairs, 2, H, 2, 64).sum(-1).max())
        p = torch.softmax(s, 1)
        L = lam[:, None]
        w = p[..., 0:1] - L * p[..., 1:2]
        wa = p[..., 0:1] + L.abs() * p[..., 1:2]
        c = 4 * 66 * 2.0 ** -24 * size + (2.0 ** -20 if self.dtype == torch.float16 else 2.0 ** -17)
        self.value = {"o": (w * v).sum(1), "dv": w * do[:, None]}
        # The forward pass's weights are 2^(s - m), m at most the row's maximum: the
        # largest is 1 or more, and both halves of each end at 2^-25, so after the
        # division by their sum each is off by 2^-25 at most, in either map.
        floor = 2.0 ** -25 * (1 + L.abs()) if self.dtype == torch.float16 else 0.0 * L
        self.size = {"o": ((c * wa + floor) * v.abs()).sum(1), "dv": c * wa * do[:, None].abs()}
        self.pairs = pairs

    def check(self, name, got):
        got = got.double()[:self.pairs] if name == "o" else got.double()[self.pairs:]
        want, half = self.value[name], torch.finfo(self.dtype).eps / 2
        least = 2.0 ** -25 if self.dtype == torch.float16 else 2.0 ** -134
        bound = want.abs() * half + least + self.size[name] * (1 + half)
        err = (got.view(want.shape) - want).abs()
        assert bool((err <= bound).all()), f"{name}: {float((err / bound).max()):.3g} times its bound"


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("edges", [20_000, 100_003, 300_001])
def test_rows_of_very_many_edges(gpu, edges, dtype):
    """One row attends every node, its weights 2^-14 to 2^-18 and all alike (logits
    within 2^-3); v.do and k have means, so that dq is the difference of two large
    sums.  dq, dlam and the nodes' dv in 64 bits."""
    from fused3s_amd.torch_ops import TorchGraph
    n, row = edges, edges // 2
    gen = torch.Generator(device="cuda").manual_seed(edges)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    rp = np.zeros(n + 1, np.int32)
    rp[row + 1:] = n
    graph = TorchGraph(rp, np.arange(n, dtype=np.int32), heads=1)
    q, k, v, do = (rand(n, 1, 128) * 0.25 for _ in range(4))
    x = [t.to(dtype) for t in (q * 0.1, k + 1.0, v + 0.5, do + 0.5)]
    lam = torch.tensor([0.25], device="cuda")
    got = step(graph, x[0], x[1], x[2], lam, x[3], 0.125)
    half = torch.finfo(dtype).eps / 2
    q, k, v, do = (t.double()[:, 0] for t in x)
    split = 2.0 ** -20 if dtype == torch.float16 else 2.0 ** -17
    total, dv, dva = torch.zeros((), device="cuda").double(), 0.0, 0.0
    g, ga = v @ do[row], v.abs() @ do[row].abs()
    for m, factor in ((0, 1.0), (1, -0.25)):
        at = slice(64 * m, 64 * m + 64)
        s = (k[:, at] @ q[row, at]) * 0.125
        p = torch.softmax(s, 0)
        D = (p * g).sum()
        want = 0.125 * factor * ((p * (g - D)) @ k[:, at])
        # logits: 66 half-steps of their sizes; g: 2^-16; weights: split
        c = split + 4 * 66 * 2.0 ** -24 * float((k[:, at].abs() @ q[row, at].abs()).max()) + 2.0 ** -16
        bound = 0.125 * abs(factor) * c * ((p * (ga + (p * ga).sum())) @ k[:, at].abs())
        bound = bound + half * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        err = (got["dq"][row, 0, at].double() - want).abs()
        assert bool((err <= bound).all()), f"dq {m}: {float((err / bound).max()):.3g} times its bound"
        dv, dva = dv + factor * p, dva + abs(factor) * p
        if m:
            assert abs(float(got["dlam"]) + float(D)) <= c * float((p * ga).sum())
    want = dv[:, None] * do[row]
    bound = c * dva[:, None] * do[row].abs() + half * want.abs() + 2.0 ** -25 * (
        dtype == torch.float16)
    err = (got["dv"][:, 0].double() - want).abs()
    assert bool((err <= bound).all()), f"dv: {float((err / bound).max()):.3g} times its bound"


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("size", [300.0, 1500.0, 3500.0])
@pytest.mark.parametrize("n", [60, 6000])
def test_logits_past_two_to_the_24(gpu, n, size, dtype):
    """One-hot maps whose logits are past float32's whole numbers: log-sum-exps are
    off by whole units there, weights finite all the same (up to logits of 2^26,
    past which the forward pass's own are not)."""
    from fused3s_amd.torch_ops import TorchGraph
    H = 3
    rp = np.arange(0, 2 * n + 1, 2, dtype=np.int32)      # row i: i and i + 1
    ci = np.sort(np.stack([np.arange(n), (np.arange(n) + 1) % n], 1), 1).reshape(-1).astype(np.int32)
    graph = TorchGraph(rp, ci, heads=H)
    gen = torch.Generator(device="cuda").manual_seed(n)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q = (size * (1 + 0.01 * rand(n, H, 128).clamp(-3, 3)) / 1.05).to(dtype)
    k = q * torch.linspace(0.1, 1.0, n, device="cuda").roll(n // 3)[:, None, None].to(dtype)
    lam = torch.tensor([0.0, 0.5, -2.0], device="cuda")
    x = q, k, rand(n, H, 128).to(dtype), lam, rand(n, H, 128).to(dtype)
    got = step(graph, *x, 0.125)
    for name, t in got.items():
        assert torch.isfinite(t).all(), name
    i = torch.arange(n, device="cuda")
    logit = lambda j: (q.double() * k[j].double()).view(n, H, 2, 64).sum(-1) * 0.125
    a, b = logit(i), logit((i + 1) % n)
    # o: where the two logits are further apart than their roundings (66 half-steps)
    # and 40, the larger's value alone, (1 - lam) of it where both maps agree
    far = ((a - b).abs() > 40 + 66 * 2.0 ** -24 * (a.abs() + b.abs())).all(-1).all(-1)
    same = (a > b)[..., 0] == (a > b)[..., 1]
    won = torch.where((a > b)[..., 0, None], x[2].double(), x[2].double()[(i + 1) % n])
    want = (1 - lam.double())[:, None] * won
    at = far[:, None] & same
    half = torch.finfo(dtype).eps / 2
    bound = half * want.abs() + 2.0 ** -20 * (1 + lam.double().abs())[:, None] * won.abs() + 2.0 ** -25
    assert ((got["o"].double() - want).abs() <= bound)[at].all() and int(at.sum()) > n
