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
