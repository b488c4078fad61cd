"""linear_cross_entropy where its exponents are largest: logits near float32's end, and rows
whose loss is near 0, on each of its routes."""
from __future__ import annotations

import pytest
import torch

from test_gpu_loss import inputs, step

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
# few classes in registers; classes streamed past; tiles; tiles of ragged rows; padded copies
ROUTES = [(64, 47), (64, 65), (256, 2049), (512, 65), (512, 2049), (301, 130), (41, 9000)]


@pytest.mark.parametrize("least", [False, True], ids=["", "others-least"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("K,V", ROUTES)
def test_bias_of_the_largest_value(gpu, K, V, dtype, reduction, least):
    """One class whose bias is the type's largest value: it is the softmax.  (bfloat16's,
    times log2(e), is past float32.)  With every other at the type's lowest, the difference
    of two logits is past it too."""
    n, top = 1000, V // 2
    _, _, b, t, _ = inputs(n, K, V, dtype, 3, ignored=0.0)
    gen = torch.Generator(device="cuda").manual_seed(K + V)
    # (whole numbers: every pass's logits are the same)
    whole = lambda *s: torch.randint(-1, 2, s, generator=gen, device="cuda").to(dtype)
    x, w = whole(n, K), whole(V, K)
    t[::3] = top
    if least:
        t[:] = top
        b[:] = torch.finfo(dtype).min
    b[top] = torch.finfo(dtype).max
    dloss = torch.ones(() if reduction == "mean" else n, device="cuda")
    got = step(x, w, b, t, dloss, reduction)
    z = x.double() @ w.double().t().contiguous() + b.double()
    others = z.clone()
    others[:, top] = -float("inf")
    assert float((z[:, top] - others.amax(1)).min()) > 1000   # (exp(-1000) is 0)
    want = z[:, top] - z.gather(1, t[:, None])[:, 0]
    if reduction == "mean":
        want = want.mean()
    else:
        assert not got["loss"][t == top].any()
    # float32 sums of K + 1 products each
    size = z.abs().amax() * (K + 8) * 2.0 ** -24
    assert bool(((got["loss"].double() - want).abs() <= size * (t != top).any()).all())
    # dz is +1 at top, -1 at the target: a power of two in the type, whatever multiplies it
    scale = 1.0 / n if reduction == "mean" else 1.0
    dz = torch.zeros(n, V, dtype=torch.float64, device="cuda")
    dz[:, top] += scale
    dz.scatter_add_(1, t[:, None], torch.full((n, 1), -scale, dtype=torch.float64, device="cuda"))
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    for name, a, c in (("dx", dz, w.double()), ("dw", dz.t().contiguous(), x.double()),
                       ("db", dz.t().contiguous(), torch.ones(n, 1, dtype=torch.float64, device="cuda"))):
        exact, size = torch.matmul(a, c), torch.matmul(a.abs(), c.abs())
        # n terms in float32, the factor's division, one rounding
        bound = half * exact.abs() * (1 + 2.0 ** -10) + tiny + (n + 8) * 2.0 ** -24 * size
        err = (got[name].double().view(exact.shape) - exact).abs()
        assert bool((err <= bound).all()), (name, float((err - bound).max()))


def test_two_classes_of_the_largest_value(gpu):
    """Two biases of the type's largest value, beside which the products are nothing: log 2."""
    from fused3s_amd.torch_ops import linear_cross_entropy
    for K, V in ROUTES:
        x, w, b, t, _ = inputs(300, K, V, torch.bfloat16, 4, ignored=0.0)
        b[[1, V - 1]] = torch.finfo(torch.bfloat16).max
        t[:] = 1
        got = linear_cross_entropy(x, w, t, b, reduction="none")
        # (log 2, in float32: its logarithm is within 2^-22)
        assert bool(((got.double() - 0.6931471805599453).abs() <= 2.0 ** -22).all()), (K, V)


@pytest.mark.parametrize("top", [100.0, 1000.0, 30_000.0])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("K,V", ROUTES)
def test_losses_near_0(gpu, K, V, dtype, top):
    """Rows whose target's logit is far above the others, or above them by whole numbers, all
    logits exact: no loss is below 0, and the loss is exact up to its exponentials and
    logarithm, however large the logits are."""
    from fused3s_amd.torch_ops import linear_cross_entropy
    n = 500
    gen = torch.Generator(device="cuda").manual_seed(K + V)
    x = torch.zeros(n, K, device="cuda")
    x[:, 0] = 1.0
    x[:, 1] = 2.0 ** -2 * torch.randint(1, 130, (n,), generator=gen, device="cuda")
    w = torch.zeros(V, K, device="cuda")
    b = torch.zeros(V, device="cuda")
    # all but the target below it by quarters of whole numbers
    t = torch.randint(V, (1,), generator=gen, device="cuda").expand(n).contiguous()
    w[:, 1] = -torch.randint(1, 5, (V,), generator=gen, device="cuda").float()
    w[t[0], 1] = 0.0
    if top <= 1000:
        b[:] = top
    else:   # (a product of two numbers of 8 bits)
        x[:, 0], w[:, 0] = 32.0, top // 128 * 4
    x, w, b = x.to(dtype), w.to(dtype), b.to(dtype)
    z = x.double() @ w.double().t().contiguous() + b.double()
    want = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
    assert float(want.min()) < 1e-6 and float(want.max()) > 1e-3
    got = linear_cross_entropy(x, w, t, b, reduction="none").double()
    assert bool((got >= 0).all()), float(got.min())
    # An exponent d log2(e) is off by 2^-23 of itself, where all but 2^-23 of the sum has d of
    # log V + 16 at most; an exponential and the logarithm by 2^-22; a lane's sum of V / 4
    # terms, and 64 more adds, by half a step of float32 each.
    bound = 2.0 ** -18 + (64 + V / 4) * 2.0 ** -24 + 2.0 ** -21 * want
    assert bool(((got - want).abs() <= bound).all()), float((got - want).abs().max())
