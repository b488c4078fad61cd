"""linear_cross_entropy and its gradient against 64 bits: every value within the type's
roundings and the bound of its 32-bit sums."""
from __future__ import annotations

import pytest
import torch

from _loss_reference import Reference

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
SHAPES = [(1, 1, 1), (1, 8, 2), (3, 5, 3), (5, 16, 7), (17, 33, 10), (64, 64, 47), (65, 128, 300),
          (100, 100, 1000), (130, 72, 129), (257, 256, 2049), (2000, 64, 40), (513, 301, 777),
          (300, 40, 20_000), (1, 512, 5000), (4100, 128, 4099), (20_011, 24, 3),
          # few classes of few inputs, 2 to 8 fragments by 1 to 4 tiles
          (3000, 256, 64), (1000, 136, 33), (257, 128, 17), (40_000, 40, 64), (130, 200, 16),
          (127, 64, 32), (129, 8, 64), (5000, 104, 48),
          # many classes of few inputs: shares of either side, one and two blocks of inputs
          (1, 64, 65), (127, 8, 128), (129, 64, 129), (3000, 120, 65), (64, 128, 9000),
          (9000, 128, 70), (333, 256, 1001)]


def inputs(n, K, V, dtype, seed, bias=True, ignored=0.2, reduction="mean"):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, w = rand(n, K).to(dtype), (2.0 * K ** -0.5 * rand(V, K)).to(dtype)
    b = (0.5 * rand(V)).to(dtype) if bias else None
    t = torch.randint(V, (n,), generator=gen, device="cuda")
    if n > 2:
        t[torch.rand(n, generator=gen, device="cuda") < ignored] = -100
    dloss = rand(n) if reduction == "none" else 1.0 + rand(()).abs()
    if dtype == torch.float16 and reduction == "mean":
        dloss = dloss * 1024.0
    return x, w, b, t, dloss


def step(x, w, b, t, dloss, reduction, ignore=-100):
    from fused3s_amd.torch_ops import linear_cross_entropy
    leaves = [None if v is None else v.detach().requires_grad_() for v in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], ignore, reduction)
    grads = torch.autograd.grad(loss, [v for v in leaves if v is not None], dloss)
    return {"loss": loss.detach(), **dict(zip(("dx", "dw", "db"), grads))}


def check(got, x, w, b, t, dloss, reduction, ignore=-100):
    ref = Reference(x, w, b, t, reduction, dloss, ignore)
    for name, v in got.items():
        ref.check(name, v)


def same(a, b):
    for name in a:
        assert torch.equal(a[name], b[name]), name


@pytest.mark.parametrize("bias", [True, False], ids=["bias", ""])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,K,V", SHAPES)
def test_step(gpu, n, K, V, dtype, reduction, bias):
    from fused3s_amd.torch_ops import linear_cross_entropy
    x = inputs(n, K, V, dtype, n + K + V, bias, reduction=reduction)
    got = step(*x, reduction)
    check(got, *x, reduction)
    same(got, step(*x, reduction))
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(*x[:2], x[3], x[2], reduction=reduction),
                           got["loss"])


@pytest.mark.parametrize("K", [136, 41, 40])
@pytest.mark.parametrize("dtype", HALF)
def test_pieces_of_the_classes(gpu, dtype, K):
    """More of dz than a piece holds, the last piece smaller and ragged."""
    x = inputs(20_000, K, 16_001, dtype, 4)
    check(step(*x, "mean"), *x, "mean")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,K,V", [(1024, 1, 8200), (1030, 7, 8191), (140_000, 63, 60),
                                   (90_001, 5, 130), (1000, 257, 8500), (1025, 301, 9001)])
def test_padded_rows(gpu, n, K, V, dtype):
    """Many rows of K inputs that are no multiple of eight, also apart from each other; each
    gradient alone."""
    from fused3s_amd.torch_ops import linear_cross_entropy
    x, w, b, t, dloss = inputs(n, K, V, dtype, n + K)
    got = step(x, w, b, t, dloss, "mean")
    check(got, x, w, b, t, dloss, "mean")
    wide = torch.full((n, K + 3), float("nan"), dtype=dtype, device="cuda")
    wide[:, 1:K + 1] = x
    for i, name in ((0, "dx"), (1, "dw")):
        leaves = [wide[:, 1:K + 1], w.cuda(), b.cuda()]
        leaves[i] = leaves[i].detach().requires_grad_()
        loss = linear_cross_entropy(leaves[0], leaves[1], t.cuda(), leaves[2])
        loss.backward(dloss.cuda())
        assert torch.equal(leaves[i].grad.cpu(), got[name].cpu()), name


def test_pieces_of_the_rows(gpu):
    """More blocks than a forward pass holds at a time."""
    from fused3s_amd.torch_ops import linear_cross_entropy
    n, V = 70_000, 17_000
    x, w, b, t, _ = inputs(n, 16, V, torch.bfloat16, 5, reduction="none")
    with torch.no_grad():
        loss = linear_cross_entropy(x, w, t, b, reduction="none")
        total = linear_cross_entropy(x, w, t, b, reduction="sum")
    for r0 in range(0, n, 10_000):
        at = slice(r0, r0 + 10_000)
        Reference(x[at], w, b, t[at], "none").check("loss", loss[at])
    assert abs(float(loss.double().sum()) - float(total)) <= 2.0 ** -23 * float(total)


@pytest.mark.parametrize("dtype", HALF)
def test_sizes_of_gradients(gpu, dtype):
    """Rows' gradients of very different sizes, and loss scales at the type's ends: what
    multiplies all of dz is not rounded with it."""
    x, w, b, t, dloss = inputs(300, 64, 500, dtype, 6, reduction="none")
    for size in (1e-30, 1e-3, 1.0, 1e4):
        g = dloss * size
        g[::3] *= 0.02
        check(step(x, w, b, t, g, "none"), x, w, b, t, g, "none")
        check(step(x, w, b, t, g.abs().max(), "mean"), x, w, b, t, g.abs().max(), "mean")
    zero = step(x, w, b, t, torch.zeros(300, device="cuda"), "none")
    assert not zero["dx"].any() and not zero["dw"].any() and not zero["db"].any()


def test_confident_and_masked_classes(gpu):
    """A loss near 0, logits in the hundreds, classes that a bias of -inf or the type's
    lowest value takes out, a row of its highest."""
    for dtype in HALF:
        x, w, b, t, dloss = inputs(200, 64, 300, dtype, 7)
        w[t.clamp(min=0)[:50]] = (8 * x[:50].float() / 8).to(dtype)
        check(step(x, w, b, t, dloss, "mean"), x, w, b, t, dloss, "mean")
        out = torch.ones(300, dtype=torch.bool, device="cuda")
        out[t[t >= 0]] = False
        low = torch.where(out, torch.finfo(dtype).min, b)
        gone = torch.where(out, float("-inf"), b)
        a, c = step(x, w, low, t, dloss, "mean"), step(x, w, gone, t, dloss, "mean")
        keep = (~out).nonzero()[:, 0]
        back = torch.full((300,), -100, device="cuda")
        back[keep] = torch.arange(keep.numel(), device="cuda")
        fewer = torch.where(t >= 0, back[t.clamp(min=0)], -100)
        ref = Reference(x, w[keep], b[keep], fewer, "mean", dloss)
        for got in (a, c):
            assert not got["dw"][out].any() and not got["db"][out].any()
            for name, v in (("loss", got["loss"]), ("dx", got["dx"]), ("dw", got["dw"][keep]),
                            ("db", got["db"][keep])):
                ref.check(name, v)


def test_ignored_and_wrong_targets(gpu):
    from fused3s_amd.torch_ops import linear_cross_entropy
    x, w, b, t, dloss = inputs(100, 32, 50, torch.bfloat16, 8, reduction="none")
    t = t.clamp(min=0)
    t[10:20] = 7
    check(step(x, w, b, t, dloss, "none", ignore=7), x, w, b, t, dloss, "none", ignore=7)
    none = torch.full_like(t, -100)
    got = step(x, w, b, none, torch.ones((), device="cuda"), "mean")
    assert got["loss"].isnan() and not any(got[k].any() for k in ("dx", "dw", "db"))
    got = step(x, w, b, none, torch.ones((), device="cuda"), "sum")
    assert float(got["loss"]) == 0.0 and not any(got[k].any() for k in ("dx", "dw", "db"))
    wrong = t.clone()
    wrong[3], wrong[4], wrong[5] = 50, -1, 2**40
    got = step(x, w, b, wrong, dloss, "none")
    want = step(x, w, b, t, dloss, "none")
    bad = torch.zeros(100, dtype=torch.bool, device="cuda")
    bad[3:6] = True
    for name in ("loss", "dx"):
        assert got[name][bad].isnan().all() and torch.equal(got[name][~bad], want[name][~bad])
    assert linear_cross_entropy(x, w, wrong, b).isnan()


def test_odd_values(gpu):
    """An infinite or NaN row of x: its loss and dx; a row that does not count has neither."""
    x, w, b, t, dloss = inputs(100, 32, 50, torch.float16, 8, reduction="none")
    t = t.clamp(min=0)
    want = step(x, w, b, t, dloss, "none")
    x[7, 3], x[60, 0] = float("inf"), float("nan")
    got = step(x, w, b, t, dloss, "none")
    rest = [i for i in range(100) if i not in (7, 60)]
    for name in ("loss", "dx"):
        assert torch.equal(got[name][rest], want[name][rest]), name
        assert got[name][[7, 60]].isnan().any(-1).all() if name == "dx" else \
            not torch.isfinite(got[name][[7, 60]]).any()
    t[[7, 60]] = -100
    got = step(x, w, b, t, dloss, "none")
    assert not got["loss"][[7, 60]].any() and not got["dx"][[7, 60]].any()


def test_layouts(gpu):
    from fused3s_amd.torch_ops import linear_cross_entropy
    for dtype in HALF:
        x, w, b, t, dloss = inputs(60, 48, 70, dtype, 9, reduction="none")
        want = step(x, w, b, t, dloss, "none")
        wide = torch.zeros(60, 61, dtype=dtype, device="cuda")
        wide[:, 5:53] = x
        got = step(wide[:, 5:53], w, b, t, dloss, "none")
        check(got, x, w, b, t, dloss, "none")
        wide = torch.zeros(60, 64, dtype=dtype, device="cuda")
        wide[:, 8:56] = x
        spread = torch.zeros(120, dtype=torch.int64, device="cuda")
        spread[::2] = t
        bias = torch.zeros(141, dtype=dtype, device="cuda")
        bias[1::2] = b
        got = step(wide[:, 8:56], w.t().contiguous().t(), bias[1::2], spread[::2], dloss, "none")
        same(got, want)
        loss = linear_cross_entropy(x.view(3, 20, 48), w, t.view(3, 20), b, reduction="none")
        assert loss.shape == (3, 20) and torch.equal(loss.view(-1), want["loss"])
        assert linear_cross_entropy(x[0], w, t[0], b).dtype is torch.float32
        leaf = x.view(3, 20, 48).detach().requires_grad_()
        linear_cross_entropy(leaf, w, t.view(3, 20), b, reduction="none").sum().backward()
        ones = step(x, w, b, t, torch.ones(60, device="cuda"), "none")
        assert torch.equal(leaf.grad.view(60, 48), ones["dx"])
        got = step(x[:0], w, b, t[:0], torch.ones((), device="cuda"), "mean")
        assert got["loss"].isnan() and got["dx"].shape == (0, 48)
        assert got["dw"].shape == w.shape and not got["dw"].any() and not got["db"].any()
        assert float(step(x[:0], w, b, t[:0], torch.ones((), device="cuda"), "sum")["loss"]) == 0.0
        # only some of the gradients
        leaf = w.detach().requires_grad_()
        g, = torch.autograd.grad(linear_cross_entropy(x, leaf, t, b, reduction="none"), [leaf], dloss)
        assert torch.equal(g, want["dw"])


@pytest.mark.parametrize("K,V", [(40, 54_000_000), (264, 8_200_001)])
def test_classes_past_4_gib(gpu, K, V):
    """Every class but some at both ends and between has a bias of -inf: the loss is theirs."""
    x, w, _, _, dloss = inputs(5, K, 8, torch.bfloat16, 11)
    w = torch.randn(V, K, device="cuda", dtype=torch.bfloat16)
    some = torch.cat([torch.arange(30), V // 2 + torch.arange(30), V - 30 + torch.arange(30)]).cuda()
    b = torch.full((V,), float("-inf"), device="cuda", dtype=torch.bfloat16)
    b[some] = torch.linspace(-1, 1, 90, device="cuda").bfloat16()
    t = torch.tensor([0, 89, 45, 60, 10], device="cuda")
    got = step(x, w, b, some[t], dloss, "mean")
    for name in ("dw", "db"):
        whole, got[name] = got[name], got[name][some]
        whole[some] = 0
        assert not whole.any(), name
        del whole
    check(got, x, w[some], b[some], t, dloss, "mean")


@pytest.mark.parametrize("n,K,V", [(54_000_000, 40, 50), (54_000_000, 40, 100), (8_200_001, 264, 70)])
def test_rows_past_4_gib(gpu, n, K, V):
    """Every row but some at both ends and between is ignored: the loss is theirs."""
    _, w, b, _, dloss = inputs(5, K, V, torch.bfloat16, 12, reduction="sum")
    x = torch.randn(n, K, device="cuda", dtype=torch.bfloat16)
    some = torch.cat([torch.arange(30), n // 2 + torch.arange(30), n - 30 + torch.arange(30)]).cuda()
    t = torch.full((n,), -100, device="cuda")
    t[some] = torch.randint(V, (90,), device="cuda")
    got = step(x, w, b, t, dloss, "sum")
    whole, got["dx"] = got["dx"], got["dx"][some]
    whole[some] = 0
    assert not whole.any()
    check(got, x[some], w, b, t[some], dloss, "sum")


def test_streams_and_capture(gpu):
    """Two calls at once, and a captured step replayed with new inputs, each replay against
    the eager result."""
    xs = [inputs(3000, 64, 1000, torch.float16, seed) for seed in (1, 2)]
    want = [step(*x, "mean") for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for s, x in zip(streams, xs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(*x, "mean"))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        same(a, b)
    x = [v.clone() for v in xs[0]]
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        out = step(*x, "mean")
    for i in (1, 0, 1):
        for v, new in zip(x, xs[i]):
            v.copy_(new)
        captured.replay()
        torch.cuda.synchronize()
        same(out, want[i])
        same(step(*xs[1 - i], "mean"), want[1 - i])


def test_refusals(gpu):
    from fused3s_amd.torch_ops import linear_cross_entropy
    x, w, b, t, _ = inputs(8, 16, 5, torch.float16, 1)
    for args in ((x.float(), w.float(), t), (x, w.bfloat16(), t), (x, w, t.int()), (x, w.cpu(), t),
                 (x, w, t.cpu()), (x, w, t, b.float()), (x, w, t.view(2, 4))):
        with pytest.raises(ValueError):
            linear_cross_entropy(*args)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        linear_cross_entropy(torch.autograd.forward_ad.make_dual(x, x), w, t)
