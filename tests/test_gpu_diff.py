"""Differential attention over a graph's edges and its gradient against 64 bits:
every value within the type's rounding and the bound of its 32-bit sums."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _diff_reference import Reference
from conftest import random_csr

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]


def directed_csr(n, degree, seed, empty=0.2):
    """Random directed edges, a share of the nodes without any of their own."""
    r = np.random.default_rng(seed)
    deg = np.where(r.random(n) < empty, 0, r.poisson(degree, n)).clip(0, n)
    cols = [np.sort(r.choice(n, d, replace=False)) for d in deg]
    rp = np.concatenate([[0], np.cumsum(deg)]).astype(np.int32)
    return rp, (np.concatenate(cols) if rp[-1] else np.zeros(0)).astype(np.int32)


def inputs(n, H, dtype, seed, scale_do=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k, v = (rand(n, H, 128).to(dtype) for _ in range(3))
    return q, k, v, 0.5 + 0.3 * rand(H), (rand(n, H, 128) * scale_do).to(dtype)


def step(graph, q, k, v, lam, do, scale):
    q, k, v, lam = (t.detach().clone().requires_grad_() for t in (q, k, v, lam))
    o = graph.diff_attention(q, k, v, lam, scale)
    dq, dk, dv, dlam = torch.autograd.grad(o, (q, k, v, lam), do)
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def packed_step(graph, q, k, v, lam, do, scale):
    n, H = q.shape[:2]
    qkv = torch.stack([q, k, v], 1).view(n, 3 * H * 128).requires_grad_()
    lam = lam.detach().clone().requires_grad_()
    o = graph.diff_attention_packed(qkv, lam, scale)
    dqkv, dlam = torch.autograd.grad(o, (qkv, lam), do)
    dq, dk, dv = dqkv.view(n, 3, H, 128).unbind(1)
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def check(got, q, k, v, lam, do, rp, ci, scale):
    ref = Reference(q, k, v, lam, do, rp, ci, scale)
    for name, t in got.items():
        ref.check(name, t)


CASES = [(1, 1, 1), (2, 1, 2), (15, 2, 1), (16, 3, 3), (17, 2, 2), (33, 30, 1), (300, 6, 3),
         (301, 40, 5), (1000, 3, 1)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,degree,H", CASES)
def test_step(gpu, n, degree, H, dtype):
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = directed_csr(n, degree, n + H)
    graph = TorchGraph(rp, ci, heads=H)
    x = inputs(n, H, dtype, n)
    got = step(graph, *x, 0.125)
    check(got, *x, rp, ci, 0.125)
    packed = packed_step(graph, *x, 0.125)
    for name in got:
        assert torch.equal(got[name], packed[name]), name
    with torch.no_grad():
        assert torch.equal(graph.diff_attention(*x[:4], 0.125), got["o"])


def test_no_edges(gpu):
    from fused3s_amd.torch_ops import TorchGraph
    rp = np.zeros(41, np.int32)
    graph = TorchGraph(rp, np.zeros(0, np.int32), heads=2)
    x = inputs(40, 2, torch.float16, 1)
    for name, t in step(graph, *x, 0.125).items():
        assert not t.any(), name


def test_no_nodes(gpu):
    from fused3s_amd.torch_ops import TorchGraph
    graph = TorchGraph(np.zeros(1, np.int32), np.zeros(0, np.int32), heads=2)
    x = inputs(0, 2, torch.float16, 1)
    got = step(graph, *x, 0.125)
    assert got["o"].shape == (0, 2, 128) and not got["dlam"].any()


@pytest.mark.parametrize("dtype", HALF)
def test_one_wave_windows_and_hubs(gpu, dtype):
    """More than 1,024 window-heads (a window per wave) and rows joined to every
    node, whose windows are split into segments and merged, in both directions."""
    from fused3s_amd.torch_ops import TorchGraph
    n, H = 5601, 3
    rp, ci = random_csr(n, 5, 3)
    rows = np.repeat(np.arange(n), np.diff(rp))
    hub = np.array([7, 2000, 2001, 5600])
    u = np.concatenate([rows, np.repeat(hub, n), np.tile(np.arange(0, n, 2), 1)])
    v = np.concatenate([ci, np.tile(np.arange(n), 4), np.full((n + 1) // 2, 40)])
    key = np.unique(u.astype(np.int64) * n + v)
    rp = np.concatenate([[0], np.cumsum(np.bincount(key // n, minlength=n))]).astype(np.int32)
    ci = (key % n).astype(np.int32)
    graph = TorchGraph(rp, ci, heads=H).prepare_backward()
    assert graph.plan.num_split > 0 and graph._reversed.num_split > 0
    x = inputs(n, H, dtype, 5)
    got = step(graph, *x, 0.125)
    check(got, *x, rp, ci, 0.125)
    again = packed_step(graph, *x, 0.125)
    for name in got:
        assert torch.equal(got[name], again[name]), name


@pytest.mark.parametrize("lam", [0.0, 1.0, -3.0, 1e6])
@pytest.mark.parametrize("scale_do", [2e4, 1e-4])
def test_magnitudes(gpu, lam, scale_do):
    """Gradients near binary16's ends and weights of any size, with every other
    row's a hundredth of its neighbours'."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(200, 6, 3)
    graph = TorchGraph(rp, ci, heads=2)
    q, k, v, _, do = inputs(200, 2, torch.float16, 3, scale_do / 4)
    v = v * 2.0 ** -6 / max(1.0, abs(lam))   # (the results stay in the type)
    do[::2] *= 0.01
    x = (q, k, v, torch.full((2,), lam, device="cuda"), do / max(1.0, abs(lam)))
    check(step(graph, *x, 0.05), *x, rp, ci, 0.05)


def test_large_logits(gpu):
    """Maps that are one-hot: the largest of logits in the hundreds."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(200, 8, 4)
    graph = TorchGraph(rp, ci, heads=1)
    q, k, v, lam, do = inputs(200, 1, torch.bfloat16, 3)
    x = (q * 8, k * 8, v, lam, do)
    check(step(graph, *x, 0.125), *x, rp, ci, 0.125)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("H,n", [(1, 200), (3, 5600)])
def test_odd_values_stay_with_their_edges(gpu, value, H, n):
    """An infinite or NaN feature reaches the rows that have an edge to its node
    (or, in the gradients, from it) and no others, which are bit for bit what they
    are without it."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = directed_csr(n, 5, 9)
    graph = TorchGraph(rp, ci, heads=H)
    x = inputs(n, H, torch.float16, 3)
    clean = step(graph, *x, 0.125)
    rows = torch.as_tensor(np.repeat(np.arange(n), np.diff(rp))).cuda()
    cols = torch.as_tensor(ci).long().cuda()
    at = int(ci[len(ci) // 2])
    sources = torch.zeros(n, dtype=torch.bool, device="cuda")
    sources[rows[cols == at]] = True          # rows with an edge to `at`
    targets = torch.zeros(n, dtype=torch.bool, device="cuda")
    targets[cols[rows == at]] = True          # nodes that `at` has an edge to
    near = targets.clone()                    # columns that share a source's row with `at`
    near[cols[sources[rows]]] = True
    own = torch.zeros_like(targets)
    own[at] = True
    for i, name in enumerate("qkv"):
        y = [t.clone() for t in x]
        y[i][at, H - 1, 5] = value
        got = step(graph, *y, 0.125)
        touched = {
            # (v: only dim 5 of o; its gradients reach every row near it)
            "o": {"q": own, "k": sources, "v": sources}[name],
            "dq": {"q": own, "k": sources, "v": sources}[name],
            "dk": {"q": targets, "k": near, "v": near}[name],
            "dv": {"q": targets, "k": near, "v": torch.zeros_like(own)}[name],
        }
        for out, rows_hit in touched.items():
            a, b = got[out], clean[out]
            assert torch.equal(a[~rows_hit], b[~rows_hit]), (name, out)
            if H > 1:
                assert torch.equal(a[:, :H - 1], b[:, :H - 1]), (name, out)
        if name == "v":
            keep = torch.arange(128, device="cuda") != 5
            assert torch.equal(got["o"][..., keep], clean["o"][..., keep])
            assert not torch.isfinite(got["o"][sources, H - 1, 5]).any()
        if name == "k" and value != value:   # (a logit of -inf is a weight of 0)
            assert not torch.isfinite(got["o"][sources, H - 1]).any()


@pytest.mark.parametrize("n", [40, 4000])
def test_logits_of_minus_infinity(gpu, n):
    """Every logit of a row -inf: NaN where one map's are, in either place, 0 where
    both maps' are, and rows with a finite logit among theirs as if it were alone."""
    from fused3s_amd.torch_ops import TorchGraph
    rp = np.arange(0, 2 * n + 1, 2, dtype=np.int32)      # row i: i and i + 1
    ci = np.sort(np.stack([np.arange(n), (np.arange(n) + 1) % n], 1), 1).reshape(-1).astype(np.int32)
    graph = TorchGraph(rp, ci, heads=1)
    q, k, v, lam, _ = inputs(n, 1, torch.float16, 5)
    q = q.abs() + 0.125
    at = {1: slice(0, 64), 2: slice(64, 128), 3: slice(0, 128)}
    for first, maps in ((4, 1), (12, 2), (20, 3)):       # nodes first .. first + 2
        k[first:first + 3, 0, at[maps]] = -float("inf")
    o = graph.diff_attention(q, k, v, lam, 0.125)
    nan = torch.isnan(o).flatten(1).all(1)
    assert nan[[4, 5, 12, 13]].all() and int(nan.sum()) == 4
    assert not o[20:22].any() and bool(torch.isfinite(o[~nan]).all())
    # row 3 attends nodes 3 and 4, node 4 by its second map only
    w = torch.softmax(torch.stack([(q[3, 0, 64:].double() * k[j, 0, 64:].double()).sum() * 0.125
                                   for j in (3, 4)]), 0)
    want = v[3, 0].double() - lam.double() * (w[0] * v[3, 0].double() + w[1] * v[4, 0].double())
    size = v[3, 0].double().abs() + lam.abs() * v[3:5, 0].double().abs().sum(0)
    # 64 products and 3 more roundings of 2^-24 in a logit of at most 16, twice
    # that as a weight's relative error, and the output's rounding
    bound = 2 * 67 * 2.0 ** -24 * 16 * size + want.abs() * 2.0 ** -11 + 2.0 ** -25
    assert bool(((o[3, 0].double() - want).abs() <= bound).all())


def test_linear_in_values_and_weights(gpu):
    """o is linear in v and in lam, so its differences there are its derivatives
    times the step, up to the rounding of the two o's."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(333, 7, 6)
    graph = TorchGraph(rp, ci, heads=2)
    q, k, v, lam, do = inputs(333, 2, torch.float16, 8)
    got = step(graph, q, k, v, lam, do, 0.125)
    with torch.no_grad():
        o = got["o"].double()
        d = do.double()
        v2 = v + torch.randn_like(v)
        o2 = graph.diff_attention(q, k, v2, lam, 0.125).double()
        delta = (d * (o2 - o)).sum()
        want = (got["dv"].double() * (v2.double() - v.double())).sum()
        # half a step of every o, o2 and dv, and 2^-14 for the 32-bit sums
        bound = 2.0 ** -11 * ((d.abs() * (o.abs() + o2.abs())).sum() + (
            got["dv"].double().abs() * (v2.double() - v.double()).abs()).sum()) * (1 + 2.0 ** -3)
        assert (delta - want).abs() <= bound
        lam2 = lam + 1.0
        o3 = graph.diff_attention(q, k, v, lam2, 0.125).double()
        delta = (d * (o3 - o)).sum((0, 2))
        bound = 2.0 ** -11 * (d.abs() * (o.abs() + o3.abs())).sum((0, 2)) * (1 + 2.0 ** -3)
        assert ((delta - got["dlam"].double()).abs() <= bound).all()


def test_layouts(gpu):
    """Rows at a distance, heads apart, a transposed view, an unaligned start, a
    gradient that is expanded: the results are those of contiguous tensors."""
    from fused3s_amd.torch_ops import TorchGraph
    n, H = 150, 2
    rp, ci = random_csr(n, 6, 2)
    graph = TorchGraph(rp, ci, heads=H)
    q, k, v, lam, do = inputs(n, H, torch.float16, 4)
    want = step(graph, q, k, v, lam, do, 0.125)
    wide = torch.zeros(n, 1000, dtype=torch.float16, device="cuda")
    wide[:, 8:264] = k.view(n, 256)
    heads_first = v.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(n * 256 + 1, dtype=torch.float16, device="cuda")
    odd[1:] = q.view(-1)
    got = graph.diff_attention(odd[1:].view(n, H, 128), wide[:, 8:264], heads_first, lam, 0.125)
    assert torch.equal(got, want["o"])
    leaf = wide.clone().requires_grad_()
    o = graph.diff_attention(q, leaf[:, 8:264], v, lam, 0.125)
    (dwide,) = torch.autograd.grad(o, leaf, do)
    assert torch.equal(dwide[:, 8:264], want["dk"].view(n, 256)) and not dwide[:, 264:].any()
    # sum(): a gradient of stride 0; weights shared by the heads: their gradients' sum
    one = lam[:1].clone().requires_grad_()
    qq = q.clone().requires_grad_()
    graph.diff_attention(qq, k, v, one.expand(H), 0.125).sum().backward()
    full = step(graph, q, k, v, lam[:1].expand(H), torch.ones_like(do), 0.125)
    assert torch.equal(qq.grad, full["dq"])
    assert torch.equal(one.grad, full["dlam"].sum(0, keepdim=True))


def test_same_tensor_thrice(gpu):
    """q, k and v one tensor: its gradient is the sum of the three."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(60, 4, 2)
    graph = TorchGraph(rp, ci, heads=1)
    x, _, _, lam, do = inputs(60, 1, torch.bfloat16, 4)
    want = step(graph, x, x, x, lam, do, 0.125)
    leaf = x.clone().requires_grad_()
    (d,) = torch.autograd.grad(graph.diff_attention(leaf, leaf, leaf, lam, 0.125), leaf, do)
    parts = [want[name].double() for name in ("dq", "dk", "dv")]
    # (autograd adds them two at a time in the type: two roundings)
    size = parts[0].abs() + parts[1].abs() + parts[2].abs()
    assert ((d.double() - sum(parts)).abs() <= 2 * 2.0 ** -8 * size).all()


def test_wide_rows(gpu):
    """Tensors past 4 GiB: 64-bit addresses give the narrow launch's bits."""
    from fused3s_amd.torch_ops import TorchGraph
    n = 70_001
    rp, ci = random_csr(n, 3, 12)
    graph = TorchGraph(rp, ci, heads=1)
    q, k, v, lam, do = inputs(n, 1, torch.float16, 4)
    want = step(graph, q, k, v, lam, do, 0.125)
    far = torch.zeros(n, 32768, dtype=torch.float16, device="cuda")
    assert far.numel() * 2 > 2**32
    got = {}
    for i, name in enumerate(("q", "k", "v")):
        x = [q, k, v]
        far[:, :128] = x[i].view(n, 128)
        x[i] = far[:, :128]
        leaves = [t.detach().requires_grad_() for t in x]
        o = graph.diff_attention(*leaves, lam, 0.125)
        grads = torch.autograd.grad(o, leaves, do)
        assert torch.equal(o, want["o"]), name
        for t, other in zip(grads, ("dq", "dk", "dv")):
            assert torch.equal(t.view(n, 1, 128), want[other]), (name, other)
    x = far[:, :128]
    x.copy_(do.view(n, 128))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = graph.diff_attention(*leaves, lam, 0.125)
    for t, other in zip(torch.autograd.grad(o, leaves, x.unsqueeze(1)), ("dq", "dk", "dv")):
        assert torch.equal(t, want[other]), other


def test_streams_and_overlap(gpu):
    """Calls of one graph on several streams at once."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(3000, 8, 2)
    graph = TorchGraph(rp, ci, heads=2)
    xs = [inputs(3000, 2, torch.float16, s) for s in range(4)]
    want = [step(graph, *x, 0.125) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [None] * len(xs)
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(graph, *xs[i], 0.125)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for name in b:
            assert torch.equal(a[name], b[name]), name


def test_capture(gpu):
    """A step captured into a graph and replayed on new inputs, eager work in
    between."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(5000, 8, 2)
    graph = TorchGraph(rp, ci, heads=4)
    static = [t.clone() for t in inputs(5000, 4, torch.float16, 0)]
    with pytest.raises(RuntimeError, match="before the capture"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(graph, *static, 0.125)
    graph.prepare_backward()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graph, *static, 0.125)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(graph, *static, 0.125)
    for seed in range(1, 4):
        x = inputs(5000, 4, torch.float16, seed)
        for a, b in zip(static, x):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        want = step(graph, *x, 0.125)
        for name in want:
            assert torch.equal(out[name], want[name]), (seed, name)


def test_reverse_csr(gpu):
    """The reversed plan's source: rows of the transposed matrix, any order."""
    from fused3s_amd import _lib
    for n, degree in ((1, 1), (50, 0.5), (3000, 9)):
        rp, ci = directed_csr(n, degree, n)
        drp, dci = torch.as_tensor(rp).cuda(), torch.as_tensor(ci).cuda()
        orp = torch.full((n + 2,), -7, dtype=torch.int32, device="cuda")
        oci = torch.full((len(ci) + 1,), -7, dtype=torch.int32, device="cuda")
        assert _lib.hip().f3s_reverse_csr(drp.data_ptr(), dci.data_ptr() if len(ci) else None, n,
                                          len(ci), orp.data_ptr(), oci.data_ptr(),
                                          torch.cuda.current_stream().cuda_stream) == 0
        orp, oci = orp.cpu().numpy(), oci.cpu().numpy()
        assert orp[n + 1] == -7 and oci[len(ci)] == -7
        rows = np.repeat(np.arange(n), np.diff(rp))
        assert np.array_equal(orp[:n + 1], np.concatenate([[0], np.cumsum(np.bincount(ci, minlength=n))]))
        for j in range(n):
            assert np.array_equal(np.sort(oci[orp[j]:orp[j + 1]]), rows[ci == j])


def test_refusals(gpu):
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(50, 4, 2)
    graph = TorchGraph(rp, ci, heads=2)
    q, k, v, lam, _ = inputs(50, 2, torch.float16, 4)
    call = graph.diff_attention
    for bad in (q.float(), q.cpu(), q[:49], q[:, :1]):
        with pytest.raises(ValueError):
            call(bad, k, v, lam)
    with pytest.raises(ValueError, match="of one type"):
        call(q, k.bfloat16(), v, lam)
    for bad in (lam[:1], lam.double(), lam.cpu(), lam.half()):
        with pytest.raises(ValueError, match="lam"):
            call(q, k, v, bad)
    with pytest.raises(ValueError, match="qkv must have shape"):
        graph.diff_attention_packed(q.view(50, 256), lam)
    with pytest.raises(ValueError, match="masked"):
        TorchGraph(rp, ci, heads=2, masked=False).diff_attention(q, k, v, lam)
    # twice differentiable it is not
    leaf = q.clone().requires_grad_()
    o = call(leaf, k, v, lam)
    (d,) = torch.autograd.grad(o.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), leaf)
