"""Edge attention (capped scores, a bias by distance) and its gradient against 64 bits:
every value within the type's rounding and the bound of its 32-bit sums."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _edge_reference import Reference
from conftest import random_csr
from test_gpu_diff import directed_csr

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
# (cap, dims of the positions): neither, each, both
BIAS = [(None, 0), (1.5, 0), (None, 1), (30.0, 2), (2.0, 3)]


def inputs(n, H, dtype, seed, dims=0, scale_do=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x = {name: rand(n, H, 64).to(dtype) for name in ("q", "k", "v")}
    x["do"] = (rand(n, H, 64) * scale_do).to(dtype)
    if dims:
        x["positions"] = 3 * rand(n, dims) if dims > 1 else 3 * rand(n)
        x["slopes"] = 0.5 + 0.5 * rand(H)
    return x


def bias_of(x, cap):
    return {"cap": cap, "positions": x.get("positions"), "slopes": x.get("slopes")}


def step(graph, x, scale=0.125, cap=None):
    leaves = {name: x[name].detach().clone().requires_grad_()
              for name in ("q", "k", "v", "slopes") if name in x}
    o = graph.edge_attention(leaves["q"], leaves["k"], leaves["v"], scale, cap, x.get("positions"),
                             leaves.get("slopes"))
    grads = torch.autograd.grad(o, list(leaves.values()), x["do"])
    return {"o": o.detach(), **{"d" + name: g for name, g in zip(leaves, grads)}}


def packed_step(graph, x, scale=0.125, cap=None):
    n, H = x["q"].shape[:2]
    qkv = torch.stack([x["q"], x["k"], x["v"]], 1).view(n, 3 * H * 64).requires_grad_()
    slopes = x["slopes"].detach().clone().requires_grad_() if "slopes" in x else None
    o = graph.edge_attention_packed(qkv, scale, cap, x.get("positions"), slopes)
    grads = torch.autograd.grad(o, [qkv] + ([] if slopes is None else [slopes]), x["do"])
    dq, dk, dv = grads[0].view(n, 3, H, 64).unbind(1)
    got = {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    return got if slopes is None else {**got, "dslopes": grads[1]}


def check(got, x, rp, ci, scale=0.125, cap=None):
    ref = Reference(x["q"], x["k"], x["v"], x["do"], rp, ci, scale, **bias_of(x, cap))
    assert set(got) == set(ref.value)
    for name, t in got.items():
        ref.check(name, t)


def same(a, b):
    for name in a:
        assert torch.equal(a[name], b[name]), name


CASES = [(1, 1, 1), (2, 1, 2), (15, 2, 1), (16, 3, 3), (17, 2, 2), (33, 30, 1), (300, 6, 3),
         (301, 40, 5), (1000, 3, 1)]


@pytest.mark.parametrize("cap,dims", BIAS)
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,degree,H", CASES)
def test_step(gpu, n, degree, H, dtype, cap, dims):
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = directed_csr(n, degree, n + H)
    graph = TorchGraph(rp, ci, heads=H)
    x = inputs(n, H, dtype, n, dims)
    got = step(graph, x, cap=cap)
    check(got, x, rp, ci, cap=cap)
    same(got, packed_step(graph, x, cap=cap))
    with torch.no_grad():
        assert torch.equal(graph.edge_attention(x["q"], x["k"], x["v"], 0.125, **bias_of(x, cap)),
                           got["o"])


def test_no_edges_and_no_nodes(gpu):
    from fused3s_amd.torch_ops import TorchGraph
    for n in (40, 20_000):
        graph = TorchGraph(np.zeros(n + 1, np.int32), np.zeros(0, np.int32), heads=2)
        for name, t in step(graph, inputs(n, 2, torch.float16, 1, 2), cap=5.0).items():
            assert not t.any(), name
    graph = TorchGraph(np.zeros(1, np.int32), np.zeros(0, np.int32), heads=2)
    got = step(graph, inputs(0, 2, torch.float16, 1, 1))
    assert got["o"].shape == (0, 2, 64) and not got["dslopes"].any()


def hub_csr(n, degree, seed):
    """Rows joined to every node, in both directions, among others."""
    rp, ci = random_csr(n, degree, seed)
    rows = np.repeat(np.arange(n), np.diff(rp))
    hub = np.array([7, n // 3, n // 3 + 1, n - 1])
    u = np.concatenate([rows, np.repeat(hub, n), np.arange(0, n, 2)])
    v = np.concatenate([ci, np.tile(np.arange(n), 4), np.full((n + 1) // 2, 40)])
    key = np.unique(u.astype(np.int64) * n + v)
    rp = np.concatenate([[0], np.cumsum(np.bincount(key // n, minlength=n))]).astype(np.int32)
    return rp, (key % n).astype(np.int32)


@pytest.mark.parametrize("cap,dims", [(None, 0), (2.0, 1), (30.0, 3)])
@pytest.mark.parametrize("dtype", HALF)
def test_one_wave_windows_and_hubs(gpu, dtype, cap, dims):
    """More than 1,024 window-heads (a window per wave) and rows joined to every node,
    whose windows are split into segments and merged, in both directions."""
    from fused3s_amd.torch_ops import TorchGraph
    n, H = 5601, 3
    rp, ci = hub_csr(n, 5, 3)
    graph = TorchGraph(rp, ci, heads=H).prepare_backward()
    assert graph.plan.num_split > 0 and graph._reversed.num_split > 0
    x = inputs(n, H, dtype, 5, dims)
    got = step(graph, x, cap=cap)
    check(got, x, rp, ci, cap=cap)
    same(got, packed_step(graph, x, cap=cap))


@pytest.mark.parametrize("n,degree,H", [(17_000, 3, 1), (9000, 4, 2), (40, 2, 64)])
def test_many_windows(gpu, n, degree, H):
    """Scheduled plans (past 1,024 window-heads), and 64 heads."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = directed_csr(n, degree, 8)
    x = inputs(n, H, torch.bfloat16, 5, 2)
    graph = TorchGraph(rp, ci, heads=H)
    got = step(graph, x, cap=10.0)
    check(got, x, rp, ci, cap=10.0)
    same(got, step(graph, x, cap=10.0))


@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("scale_do", [2e4, 1e-4])
def test_magnitudes(gpu, scale_do, cap):
    """Gradients near binary16's ends, with every other row's a hundredth of its
    neighbours'."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(200, 6, 3)
    graph = TorchGraph(rp, ci, heads=2)
    x = inputs(200, 2, torch.float16, 3, 3, scale_do / 4)
    x["v"] = x["v"] * 2.0 ** -6   # (the results stay in the type)
    x["do"][::2] *= 0.01
    check(step(graph, x, 0.05, cap), x, rp, ci, 0.05, cap)


@pytest.mark.parametrize("scale,cap", [(1.0, None), (-0.5, None), (0.0, None), (-0.125, 4.0),
                                       (1.0, 0.01), (1.0, 500.0), (0.0, 2.0)])
def test_scales_and_caps(gpu, scale, cap):
    """One-hot rows, negative and zero scales, caps that all scores reach or none does."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(200, 8, 4)
    graph = TorchGraph(rp, ci, heads=1)
    x = inputs(200, 1, torch.bfloat16, 3, 1)
    check(step(graph, x, scale, cap), x, rp, ci, scale, cap)


def test_far_positions(gpu):
    """Distances that leave one neighbour, none of them (all far, equally) or far larger
    slopes; negative slopes."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(300, 8, 4)
    graph = TorchGraph(rp, ci, heads=2)
    for dims, factor in ((1, 1e3), (3, 1e3), (2, 1e-20), (1, 1e-30)):
        x = inputs(300, 2, torch.bfloat16, 3, dims)
        x["positions"] = x["positions"] * factor
        x["slopes"] = torch.tensor([1.0, -0.25], device="cuda")
        check(step(graph, x), x, rp, ci)


@pytest.mark.parametrize("n,H", [(250, 1), (4000, 5)])
def test_infinite_scores(gpu, n, H):
    """Positions infinitely far take their nodes out, as no edge would; a row with no
    other neighbour is 0."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(n, 5, 4, self_loops=False)
    x = inputs(n, H, torch.float16, 3, 1)
    x["slopes"] = x["slopes"].abs() + 0.1
    far = torch.zeros(n, dtype=torch.bool)
    far[::7] = True
    rows = np.repeat(np.arange(n), np.diff(rp))
    keep = ~far.numpy()[ci] & ~far.numpy()[rows]
    rp2 = np.concatenate([[0], np.cumsum(np.bincount(rows[keep], minlength=n))]).astype(np.int32)
    near = TorchGraph(rp2, ci[keep], heads=H)
    with torch.no_grad():
        want = near.edge_attention(x["q"], x["k"], x["v"], 0.125, **bias_of(x, None))
        x["positions"][far.cuda()] = float("inf")
        got = TorchGraph(rp, ci, heads=H).edge_attention(x["q"], x["k"], x["v"], 0.125,
                                                         **bias_of(x, None))
    finite = ~far.cuda()
    assert torch.isfinite(got[finite]).all()
    # (the same weights in chunks that may differ: a step of the type and 2^-20 of v's)
    err = (got[finite].double() - want[finite].double()).abs()
    assert bool((err <= 2.0 ** -10 * want[finite].double().abs() + 2.0 ** -17).all())


@pytest.mark.parametrize("cap,dims", [(None, 0), (3.0, 2)])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,H,hubs", [(250, 1, False), (900, 2, False), (9000, 2, False),
                                      (5601, 3, True)])
def test_odd_values_reach_their_neighbours_only(gpu, n, H, hubs, dtype, cap, dims):
    """Infinite and NaN values of one node: rows without an edge to it are as if it were
    finite."""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = hub_csr(n, 4, 9) if hubs else directed_csr(n, 4, 9)
    graph = TorchGraph(rp, ci, heads=H)
    x = inputs(n, H, dtype, 5, dims)
    clean = step(graph, x, cap=cap)
    rows = np.repeat(np.arange(n), np.diff(rp))
    bad = np.array([3, n // 2])
    for name in ("v", "k", "q", "do"):
        y = {key: t.clone() for key, t in x.items()}
        y[name][3, 0, 5] = float("inf")
        y[name][n // 2, H - 1, 63] = float("nan")
        got = step(graph, y, cap=cap)
        # one edge away in each direction, and two: D of a row reaches its neighbours' dk
        hit = np.zeros(n, bool)
        hit[bad] = True
        one = hit.copy()
        one[rows[hit[ci]]] = True      # rows with an edge to it
        two = one.copy()
        two[ci[one[rows]]] = True      # and the nodes that those have an edge to
        for key, reach in (("o", one), ("dq", one), ("dk", two), ("dv", two)):
            clear = torch.as_tensor(~reach).cuda()
            a, b = got[key][clear].double(), clean[key][clear].double()
            assert bool(torch.isfinite(a).all()), (name, key)
            size = b.abs().amax() if b.numel() else 0.0
            # (a window done edge by edge: other orders of the same sums)
            bound = 2 * torch.finfo(dtype).eps * b.abs() + 2.0 ** -13 * size
            assert bool(((a - b).abs() <= bound).all()), (name, key)
        # and where it has an edge it is seen
        if name == "v":
            direct = np.zeros(n, bool)
            direct[rows[ci == n // 2]] = True
            if direct.any():
                assert bool(got["o"][torch.as_tensor(direct).cuda(), H - 1, 63].isnan().all())


def test_strides(gpu):
    """Slices of wider tensors, other orders and misaligned ones, gradients of any
    layout."""
    from fused3s_amd.torch_ops import TorchGraph
    n, H = 333, 2
    rp, ci = random_csr(n, 5, 7)
    graph = TorchGraph(rp, ci, heads=H)
    x = inputs(n, H, torch.bfloat16, 2, 2)
    want = step(graph, x, cap=5.0)
    wide = torch.zeros(n, H * 64 + 24, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:8 + H * 64] = x["q"].view(n, -1)
    heads_first = x["k"].transpose(0, 1).contiguous().transpose(0, 1)
    shifted = torch.zeros(n * H * 64 + 1, dtype=torch.bfloat16, device="cuda")
    shifted[1:] = x["v"].reshape(-1)
    positions = torch.zeros(n, 4, device="cuda")
    positions[:, 1:3] = x["positions"]
    slopes = torch.zeros(2 * H, device="cuda")
    slopes[::2] = x["slopes"]
    do = x["do"].transpose(0, 2).contiguous().transpose(0, 2)
    y = {"q": wide[:, 8:8 + H * 64], "k": heads_first, "v": shifted[1:].view(n, H, 64), "do": do}
    leaves = [y[name].detach().requires_grad_() for name in ("q", "k", "v")]
    s = slopes[::2].detach().requires_grad_()
    o = graph.edge_attention(*leaves, 0.125, 5.0, positions[:, 1:3], s)
    grads = torch.autograd.grad(o, leaves + [s], y["do"])
    got = {"o": o.detach(), "dq": grads[0].view(n, H, 64), "dk": grads[1], "dv": grads[2],
           "dslopes": grads[3]}
    same(got, want)


def test_past_32_bit_offsets(gpu):
    """Rows so far apart that the tensors end past 4 GiB: the same bits as side by side."""
    from fused3s_amd.torch_ops import TorchGraph
    n, H = 36_000, 1
    rp, ci = random_csr(n, 4, 7)
    graph = TorchGraph(rp, ci, heads=H)
    x = inputs(n, H, torch.float16, 2, 1)
    want = packed_step(graph, x, cap=5.0)
    qkv = torch.empty(n, 64_000, dtype=torch.float16, device="cuda")[:, :192]
    qkv.copy_(torch.stack([x["q"], x["k"], x["v"]], 1).view(n, 192))
    qkv.requires_grad_()
    o = graph.edge_attention_packed(qkv, 0.125, 5.0, x["positions"], x["slopes"])
    do = torch.empty(n, 64_000, dtype=torch.float16, device="cuda")[:, :64]
    do.copy_(x["do"].view(n, 64))
    g, = torch.autograd.grad(o, [qkv], do.unsqueeze(1))
    assert torch.equal(o, want["o"])
    for i, name in enumerate(("dq", "dk", "dv")):
        assert torch.equal(g[:, 64 * i:64 * i + 64], want[name].view(n, 64)), name


def test_streams_and_capture(gpu):
    """Two calls at once on streams of their own, and a captured step replayed with new
    inputs, each replay against the eager result."""
    from fused3s_amd.torch_ops import TorchGraph
    n, H = 20_000, 2
    rp, ci = hub_csr(n, 4, 3)
    graph = TorchGraph(rp, ci, heads=H).prepare_backward()
    xs = [inputs(n, H, torch.float16, seed, 2) for seed in (1, 2)]
    want = [step(graph, x, cap=9.0) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for s, x in zip(streams, xs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(graph, x, cap=9.0))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        same(a, b)
    x = {key: t.clone() for key, t in xs[0].items()}
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        out = step(graph, x, cap=9.0)
    for i in (1, 0, 1):
        for key in x:
            x[key].copy_(xs[i][key])
        captured.replay()
        torch.cuda.synchronize()
        same(out, want[i])
        same(step(graph, xs[1 - i], cap=9.0), want[1 - i])


def test_refusals(gpu):
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = random_csr(40, 3, 1)
    graph = TorchGraph(rp, ci, heads=2)
    x = inputs(40, 2, torch.float16, 1, 2)
    q, k, v, pos, slopes = (x[name] for name in ("q", "k", "v", "positions", "slopes"))
    for bad in (dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")),
                dict(positions=pos), dict(slopes=slopes),
                dict(positions=pos[:39], slopes=slopes), dict(positions=pos.double(), slopes=slopes),
                dict(positions=torch.zeros(40, 4, device="cuda"), slopes=slopes),
                dict(positions=torch.zeros(40, 0, device="cuda"), slopes=slopes),
                dict(positions=pos.cpu(), slopes=slopes), dict(positions=pos, slopes=slopes[:1]),
                dict(positions=pos, slopes=slopes.half())):
        with pytest.raises(ValueError):
            graph.edge_attention(q, k, v, 0.125, **bad)
    with pytest.raises(RuntimeError, match="detach"):
        graph.edge_attention(q, k, v, 0.125, positions=pos.clone().requires_grad_(), slopes=slopes)
    for bad in ((q.float(), k, v), (q, k.bfloat16(), v), (q, k, v[:, :1]), (q.cpu(), k, v)):
        with pytest.raises(ValueError):
            graph.edge_attention(*bad)
    with pytest.raises(ValueError, match="masked"):
        TorchGraph(rp, ci, heads=2, masked=False).edge_attention(q, k, v)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        graph.edge_attention(torch.autograd.forward_ad.make_dual(q, q), k, v)
