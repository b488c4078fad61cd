"""The cross entropy of a linear classifier and its gradient in 64 bits, by the formula,
and for every result the largest error that 32-bit sums, one rounding of the logits'
gradient and one of the result leave."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24


class Reference:
    def __init__(self, x, w, b, target, reduction, dloss=None, ignore=-100):
        dtype = x.dtype
        half = torch.finfo(dtype).eps / 2
        least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
        n, K = x.shape
        V = w.shape[0]
        counted = target != ignore
        many = int(counted.sum())
        x, w = x.double(), w.double()
        bias = torch.zeros(V, dtype=torch.float64, device=x.device) if b is None else b.double()
        mm = torch.matmul
        t = lambda a: a.t().contiguous()
        z = mm(x, t(w)) + bias
        # a logit: at most K + 4 half-steps of the sum of its products' sizes
        ez = (K + 4) * U * (mm(x.abs(), t(w.abs())) + bias.abs())
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(1, keepdim=True)
        lse = top + torch.log(total)
        at = target.clamp(min=0)[:, None]
        value = torch.where(counted, (lse - z.gather(1, at))[:, 0], 0.0)
        # the exponents' and log-sum-exps' own roundings, by their sizes; sums of V
        # terms, 64 in a block, V / 512 blocks in a chain
        err = ez.amax(1) + 2.0 ** -22 * (z.abs().amax(1) + math.log(V) + 1)
        el = torch.where(counted, 2 * err + (64 + V / 512) * U + 2.0 ** -20
                         + 2.0 ** -22 * (value + math.log(V)), 0.0)
        div = {"mean": max(many, 1), "sum": 1, "none": 1}[reduction]
        if reduction == "none":
            self.value, self.bound = {"loss": value}, {"loss": el + U * value}
        else:
            s = value.sum() / div
            self.value = {"loss": s}
            self.bound = {"loss": el.sum() / div + 2 * U * s.abs()}
        if dloss is None:
            return
        g = (dloss.double().expand(n) * counted / div)[:, None]
        p = e / total
        d = p.clone()
        d.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
        ep = p * (4 * err[:, None] + (64 + V / 512) * U + 2.0 ** -19) + 2 * U * d.abs()
        dz, edz = d * g, ep * g.abs()
        # rounded to the type (binary16: times 2^14 over what multiplies all of it)
        small = least * 2.0 ** -14 * 2 * float(g.abs().max()) if dtype == torch.float16 else least
        er = edz + half * (dz.abs() + edz) + small
        round_ = lambda v, size: size + half * (v.abs() * (1 + 2.0 ** -10) + size) + least
        dx, dw, db = mm(dz, w), mm(t(dz), x), dz.sum(0)
        self.value.update(dx=dx, dw=dw, db=db)
        self.bound.update(
            dx=round_(dx, mm(er, w.abs()) + (V + 8) * U * mm(dz.abs() + er, w.abs())),
            dw=round_(dw, mm(t(er), x.abs()) + (n + 8) * U * mm(t(dz.abs() + er), x.abs())),
            db=round_(db, edz.sum(0) + (n + 8) * U * (dz.abs() + edz).sum(0)))

    def check(self, name, got):
        want, bound = self.value[name], self.bound[name]
        assert got.shape == want.shape, name
        got = got.detach()
        # (a value past the type's largest is rounded to infinity, of its sign)
        most = torch.finfo(got.dtype).max
        past = got.isinf() & (got.double() * want > 0) & (want.abs() + bound > most)
        assert bool((torch.isfinite(got) | past).all()), name
        err = torch.where(past, 0.0, (got.double() - want).abs())
        worst = (err / bound.clamp_min(1e-300)).max() if err.numel() else 0.0
        assert bool((err <= bound).all()), f"{name}: {float(worst):.3g} times its bound"
