"""Layer norm and its gradient in 64 bits, by the formula, and for every result the
largest error that 32-bit sums and one rounding to the type leave."""
from __future__ import annotations

import torch

U = 2.0 ** -24
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}


class Reference:
    def __init__(self, x, w, b, dy, eps):
        n, C = x.shape
        self.types = {"y": x.dtype, "dx": x.dtype, "dw": None if w is None else w.dtype,
                      "db": None if b is None else b.dtype}
        x, dy = x.double(), dy.double()
        w = torch.ones(C, device=x.device).double() if w is None else w.double()
        b = torch.zeros(C, device=x.device).double() if b is None else b.double()
        mean = lambda t: t.mean(1, keepdim=True)
        m = mean(x)
        c = x - m
        var = mean(c * c)
        r = (var + eps) ** -0.5
        h = c * r
        dh = dy * w
        s0, s1 = mean(dh), mean(dh * h)
        inner = dh - s0 - h * s1
        self.value = {"y": h * w + b, "dx": r * inner, "dw": (dy * h).sum(0), "db": dy.sum(0)}
        # A sum of N values is off by at most (the longest chain of additions) half-steps
        # of the sum of their sizes: 16 of a lane, 6 of a wave, 16 of a workgroup; a lane
        # of a row that is read in turns has C / 1024, one of a column n / 64 at most.
        d = 40 + C / 1024
        em = (d + 2) * U * mean(x.abs())                  # of m
        ec = em + U * c.abs()
        ev = (d + 4) * U * var + 2 * em * mean(c.abs()) + em * em
        er = 0.6 * ev / (var + eps) + 6 * U               # of r, relative (root, quotient)
        eh = r * ec + h.abs() * (er + 2 * U)
        e0 = (d + 3) * U * mean(dh.abs())
        e1 = (d + 4) * U * mean((dh * h).abs()) + mean(dh.abs() * eh)
        dn = d + n / 64
        self.size = {
            "y": w.abs() * eh + 2 * U * ((h * w).abs() + b.abs()),
            "dx": r * (4 * U * (dh.abs() + s0.abs() + (h * s1).abs()) + e0 + h.abs() * e1
                       + eh * s1.abs()) + (er + 2 * U) * r * inner.abs(),
            "dw": dn * U * (dy * h).abs().sum(0) + (dy.abs() * eh).sum(0),
            "db": dn * U * dy.abs().sum(0),
        }

    def check(self, name, got):
        want, half = self.value[name], torch.finfo(self.types[name]).eps / 2
        assert got.dtype is self.types[name] and got.shape == want.shape, name
        bound = (want.abs() * half * (1 + 2.0 ** -10) + LEAST[got.dtype]
                 + self.size[name] * (1 + half))
        assert bool(torch.isfinite(got).all()), name
        err = (got.detach().double() - want).abs()
        worst = (err / bound).max() if err.numel() else 0.0
        assert bool((err <= bound).all()), f"{name}: {float(worst):.3g} times its bound"
