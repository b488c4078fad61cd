"""Differential attention over a graph's edges in 64 bits, dense: one [n, n]
matrix per map and head, rows without edges 0; its gradient by the formula, and
the sizes that rounding errors are proportional to."""
from __future__ import annotations

import torch


def adjacency(n, row_ptr, col_idx):
    a = torch.zeros(n, n, dtype=torch.bool)
    rp = torch.as_tensor(row_ptr).long()
    rows = torch.repeat_interleave(torch.arange(n), rp[1:] - rp[:-1])
    a[rows, torch.as_tensor(col_idx).long()] = True
    return a


def softmax_maps(q, k, adj, scale):
    """[2, H, n, n]: the maps' weights; q, k [n, H, 128] float64."""
    n, H = q.shape[0], q.shape[1]
    q2 = q.view(n, H, 2, 64).permute(2, 1, 0, 3)
    k2 = k.view(n, H, 2, 64).permute(2, 1, 3, 0).contiguous()
    s = torch.matmul(q2, k2) * scale
    s = s.masked_fill(~adj, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-300)


def forward(q, k, v, lam, adj, scale):
    p = softmax_maps(q, k, adj, scale)
    w = p[0] - lam.view(-1, 1, 1) * p[1]
    return torch.matmul(w, v.transpose(0, 1)).transpose(0, 1)


class Reference:
    """o, dq, dk, dv, dlam in 64 bits of 16-bit inputs, and for each the largest
    error that 32-bit sums and one rounding leave (`bound`)."""

    def __init__(self, q, k, v, lam, do, row_ptr, col_idx, scale):
        n, H = q.shape[0], q.shape[1]
        dev = q.device
        self.half = torch.finfo(q.dtype).eps / 2
        # the least that the type holds: half a subnormal step
        self.least = (2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134)
        split = 2.0 ** -22 if q.dtype == torch.float16 else 2.0 ** -17
        adj = adjacency(n, row_ptr, col_idx).to(dev)
        q, k, v, do = (t.double().view(n, H, 128) for t in (q, k, v, do))
        lam = lam.double()
        p = softmax_maps(q, k, adj, scale)
        L = lam.view(-1, 1, 1)
        w = p[0] - L * p[1]
        wa = p[0] + L.abs() * p[1]
        rows = lambda t: t.transpose(0, 1)                       # [H, n, ...]
        cols = lambda t: t.transpose(-1, -2).contiguous()
        mm = lambda a, b: rows(torch.matmul(a, b))
        V, dO = rows(v).contiguous(), rows(do).contiguous()
        g = torch.matmul(dO, cols(V))
        ga = torch.matmul(dO.abs(), cols(V.abs()))
        D = (p * g).sum(-1, keepdim=True)
        Da = (p * ga).sum(-1, keepdim=True)
        ds = torch.stack([p[0] * (g - D[0]), -L * p[1] * (g - D[1])])
        da = torch.stack([p[0] * (ga + Da[0]), L.abs() * p[1] * (ga + Da[1])])
        maps = lambda t: t.view(n, H, 2, 64).permute(2, 1, 0, 3).contiguous()
        join = lambda t: t.permute(2, 1, 0, 3).reshape(n, H, 128)
        Q, K = maps(q), maps(k)
        self.value = {
            "o": mm(w, V),
            "dq": join(torch.matmul(ds, K)) * scale,
            "dk": join(torch.matmul(cols(ds), Q)) * scale,
            "dv": mm(cols(w), dO),
            "dlam": -D[1].sum((1, 2)),
        }
        # Logits: 64 products summed in float32, at most 66 half-steps of the sum
        # of their sizes; 2^x of that, its rounding and the row's sum: 2^-20.
        logit = 66 * 2.0 ** -24 * abs(scale) * torch.matmul(
            Q.abs(), cols(K.abs())).masked_fill(~adj, 0.0).amax() if n else 0.0
        logit = float(logit)
        c = split + 4 * logit + 2.0 ** -20
        cg = c + 2.0 ** -16   # and g: 128 products (a sum, its difference from D)
        # Weights are split into halves that end at 2^-25 of a row's largest.
        floor = 2.0 ** -22
        # Float32's subnormals are not kept: a weight p below 2^-126 is 0, so p is
        # off by up to 2^-126 and p (g - D) by that times the sizes of g and D, and
        # by as much again as an operand of the second product.
        on = adj.double().expand_as(p[0])
        under = 2.0 ** -125 * on
        under_g = 2.0 ** -125 * on * (1 + ga + Da.amax(0)) if n else on
        wide = lambda t, dim: t.amax(dim, keepdim=True) * adj if n else t
        self.size = {
            "o": c * mm(wa, V.abs()) + mm(floor * wide(wa, -1) + under * (1 + L.abs()), V.abs()),
            "dq": abs(scale) * join(torch.matmul(
                cg * da + floor * wide(da, -1) + under_g * (1 + L.abs()), K.abs())),
            "dk": abs(scale) * join(torch.matmul(
                cols(cg * da + floor * wide(da, -2) + under_g * (1 + L.abs())), Q.abs())),
            "dv": mm(cols(c * wa + floor * wide(wa, -2) + under * (1 + L.abs())), dO.abs()),
            "dlam": cg * Da[1].sum((1, 2)),
        }

    def bound(self, name):
        step = 2.0 ** -24 if name == "dlam" else self.half
        least = 0.0 if name == "dlam" else self.least
        return self.value[name].abs() * step * (1 + 2.0 ** -10) + least + self.size[name] * (1 + step)

    def check(self, name, got):
        want, bound = self.value[name], self.bound(name)
        err = (got.detach().double().view(want.shape) - want).abs()
        assert bool(torch.isfinite(got).all()), name
        worst = (err / bound.clamp_min(1e-300)).max() if err.numel() else 0.0
        assert bool((err <= bound).all()), f"{name}: {float(worst):.3g} times its bound"
