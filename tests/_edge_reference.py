"""Attention over a graph's edges with capped scores and a bias by distance in 64 bits,
dense: one [n, n] matrix per head, rows without edges 0; its gradient by the formula,
and the sizes that rounding errors are proportional to."""
from __future__ import annotations

import torch

from _diff_reference import adjacency


def scores(q, k, positions, slopes, scale, cap):
    """[H, n, n] scores, their slope in scale q.k, and the [n, n] distances; q, k
    [n, H, 64] float64."""
    x = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * scale
    c = torch.ones_like(x)
    if cap:
        t = torch.tanh(x / cap)
        x, c = cap * t, 1 - t * t
    dist = None
    if positions is not None:
        p = positions.double().view(positions.shape[0], -1)
        dist = (p[:, None] - p[None]).square().sum(-1).sqrt()
        x = x - slopes.double().view(-1, 1, 1) * dist
    return x, c, dist


def softmax(s, adj):
    s = s.masked_fill(~adj, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-300)


def forward(q, k, v, slopes, positions, adj, scale, cap):
    s, _, _ = scores(q, k, positions, slopes, scale, cap)
    return torch.matmul(softmax(s, adj), v.transpose(0, 1)).transpose(0, 1)


class Reference:
    """o, dq, dk, dv, dslopes in 64 bits of 16-bit inputs, and for each the largest error
    that 32-bit sums and one rounding leave (`bound`)."""

    def __init__(self, q, k, v, do, row_ptr, col_idx, scale, cap=None, positions=None, slopes=None):
        n, H = q.shape[0], q.shape[1]
        dev = q.device
        self.half = torch.finfo(q.dtype).eps / 2
        # the least that the type holds: half a subnormal step
        self.least = 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134
        split = 2.0 ** -22 if q.dtype == torch.float16 else 2.0 ** -17
        adj = adjacency(n, row_ptr, col_idx).to(dev)
        q, k, v, do = (t.double().view(n, H, 64) for t in (q, k, v, do))
        s, c, dist = scores(q, k, positions, slopes, scale, cap)
        p = softmax(s, adj)
        rows = lambda t: t.transpose(0, 1)                       # [H, n, ...]
        cols = lambda t: t.transpose(-1, -2).contiguous()
        mm = lambda a, b: rows(torch.matmul(a, b))
        Q, K, V, dO = (rows(t).contiguous() for t in (q, k, v, do))
        g = torch.matmul(dO, cols(V))
        ga = torch.matmul(dO.abs(), cols(V.abs()))
        D = (p * g).sum(-1, keepdim=True)
        Da = (p * ga).sum(-1, keepdim=True)
        ds = p * (g - D)
        da = p * (ga + Da)
        self.value = {
            "o": mm(p, V),
            "dq": mm(ds * c, K) * scale,
            "dk": mm(cols(ds * c), Q) * scale,
            "dv": mm(cols(p), dO),
        }
        # Scores.  64 products summed in float32: at most 66 half-steps of the sum of their
        # sizes.  tanh is within 2^-20 of itself (the kernel's own bound, 3e-7, and the
        # roundings of scale / cap and cap log2(e)); a distance within 2^-21 (a difference,
        # three squares and their sum, a root), times the slope 2^-20; the score's own
        # rounding and that of what is subtracted from it, 2^-22 of the largest.
        size = abs(scale) * torch.matmul(Q.abs(), cols(K.abs()))
        x = s if dist is None else s + slopes.double().view(-1, 1, 1) * dist
        err = 66 * 2.0 ** -24 * size + 2.0 ** -20 * x.abs() + 2.0 ** -22 * s.abs()
        if dist is not None:
            err = err + 2.0 ** -20 * (slopes.double().view(-1, 1, 1) * dist).abs()
        score = float(err.masked_fill(~adj, 0.0).amax()) if n else 0.0
        e = split + 4 * score + 2.0 ** -20
        # and g, 64 products, a sum and its difference from D; c = 1 - t^2 (2^-18)
        eg = e + 2.0 ** -16
        # Weights are split into halves that end at 2^-25 of a row's largest.
        floor = 2.0 ** -22
        # Float32's subnormals are not kept: a weight p below 2^-126 is 0, so p is off by
        # up to 2^-126 and p (g - D) by that times the sizes of g and D, and by as much
        # again as an operand of the second product.
        on = adj.double().expand_as(p)
        under = 2.0 ** -125 * on
        under_g = 2.0 ** -125 * on * (1 + ga + Da.amax(0)) if n else on
        wide = lambda t, dim: t.amax(dim, keepdim=True) * adj if n else t
        self.size = {
            "o": mm(e * p + floor * wide(p, -1) + under, V.abs()),
            "dq": abs(scale) * mm(eg * da + floor * wide(da, -1) + under_g, K.abs()),
            "dk": abs(scale) * mm(cols(eg * da + floor * wide(da, -2) + under_g), Q.abs()),
            "dv": mm(cols(e * p + floor * wide(p, -2) + under), dO.abs()),
        }
        if dist is not None:
            self.value["dslopes"] = -(ds * dist).sum((1, 2))
            self.size["dslopes"] = eg * (da * dist).sum((1, 2)) + (under_g * dist).sum((1, 2))

    def bound(self, name):
        step = 2.0 ** -24 if name == "dslopes" else self.half
        least = 0.0 if name == "dslopes" else self.least
        return self.value[name].abs() * step * (1 + 2.0 ** -10) + least + self.size[name] * (1 + step)

    def check(self, name, got):
        want, bound = self.value[name], self.bound(name)
        err = (got.detach().double().view(want.shape) - want).abs()
        assert bool(torch.isfinite(got).all()), name
        worst = (err / bound.clamp_min(1e-300)).max() if err.numel() else 0.0
        assert bool((err <= bound).all()), f"{name}: {float(worst):.3g} times its bound"
