"""Differential attention where waves take their windows from a queue (some 4,096
window-heads and more), with hub windows in segments, against 64 bits; its odd values,
mended by the launch after it; calls at once and replays."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import test_gpu_diff as small
from conftest import random_csr
from test_gpu_diff import HALF, check, inputs, step

pytestmark = pytest.mark.gpu

QUEUE = 2 * 512 * 4   # units: two for each of 512 workgroups' four waves


def hub_graph(n, degree, seed):
    """Random symmetric edges, rows joined to every node and nodes that every other row
    attends, and a stretch of nodes without an edge."""
    rp, ci = random_csr(n, degree, seed)
    rows = np.repeat(np.arange(n), np.diff(rp))
    hub = np.array([7, n // 3, n // 3 + 1, n - 1])
    u = np.concatenate([rows, np.repeat(hub, n), np.arange(0, n, 2)])
    v = np.concatenate([ci, np.tile(np.arange(n), 4), np.full((n + 1) // 2, 40)])
    key = np.unique(u.astype(np.int64) * n + v)
    key = key[(key // n < 800) | (key // n >= 832)]
    rp = np.concatenate([[0], np.cumsum(np.bincount(key // n, minlength=n))]).astype(np.int32)
    return rp, (key % n).astype(np.int32)


def heads(x, got, H, rp, ci, scale):
    """Every head on its own: the reference's matrices are n by n."""
    q, k, v, lam, do = x
    for h in range(H):
        part = [t[:, h:h + 1].contiguous() for t in (q, k, v)] + [lam[h:h + 1],
                                                                 do[:, h:h + 1].contiguous()]
        check({name: t[h:h + 1] if name == "dlam" else t[:, h:h + 1] for name, t in got.items()},
              *part, rp, ci, scale)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,H", [(8900, 8), (4500, 16)])
def test_step(gpu, n, H, dtype):
    """(8,900 nodes: the library's sequence; 4,500: 282 windows, natural order.)"""
    from fused3s_amd.torch_ops import TorchGraph
    rp, ci = hub_graph(n, 5, 3)
    graph = TorchGraph(rp, ci, heads=H).prepare_backward()
    for plan in (graph._diff_plan(), graph._reversed):
        assert plan.num_items * H >= QUEUE and plan.num_split > 0
    x = inputs(n, H, dtype, 5)
    got = step(graph, *x, 0.125)
    heads(x, got, H, rp, ci, 0.125)
    for other in (step, small.packed_step):
        again = other(graph, *x, 0.125)
        for name in got:
            assert torch.equal(got[name], again[name]), name


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_odd_values_stay_with_their_edges(gpu, value):
    small.test_odd_values_stay_with_their_edges(gpu, value, 8, 9000)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_odd_values_in_segments(gpu, value):
    """A hub's window is joined from segments, some of which hold the value: its row is
    not finite, and rows of the same window without an edge to it are untouched."""
    from fused3s_amd.torch_ops import TorchGraph
    n, H = 8900, 8
    rp, ci = hub_graph(n, 5, 3)
    graph = TorchGraph(rp, ci, heads=H)
    x = inputs(n, H, torch.float16, 3)
    clean = step(graph, *x, 0.125)
    rows = torch.as_tensor(np.repeat(np.arange(n), np.diff(rp))).cuda()
    at = 5000
    hit = torch.zeros(n, dtype=torch.bool, device="cuda")
    hit[rows[torch.as_tensor(ci).cuda() == at]] = True
    assert hit[7] and hit[n // 3] and not hit[6]
    v = x[2].clone()
    v[at, 3, 9] = value
    got = step(graph, x[0], x[1], v, *x[3:], 0.125)
    assert torch.equal(got["o"][~hit], clean["o"][~hit])
    assert not torch.isfinite(got["o"][hit, 3, 9]).any()
    keep = torch.arange(128, device="cuda") != 9
    assert torch.equal(got["o"][..., keep], clean["o"][..., keep])
    assert torch.equal(got["dq"][~hit], clean["dq"][~hit])


def test_overlap_and_replay(gpu):
    """Calls of one graph on three streams at once, and a captured step replayed on new
    inputs with eager steps between: a queue belongs to its call."""
    from fused3s_amd.torch_ops import TorchGraph
    n, H = 8900, 8
    rp, ci = hub_graph(n, 5, 3)
    graph = TorchGraph(rp, ci, heads=H).prepare_backward()
    xs = [inputs(n, H, torch.bfloat16, s) for s in range(3)]
    want = [step(graph, *x, 0.125) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(2):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(step(graph, *x, 0.125))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for name in b:
                assert torch.equal(a[name], b[name]), name
    static = [t.clone() for t in xs[0]]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(graph, *static, 0.125)
    for i in (1, 2, 0, 1):
        for a, b in zip(static, xs[i]):
            a.copy_(b)
        g.replay()
        eager = step(graph, *xs[(i + 1) % 3], 0.125)
        torch.cuda.synchronize()
        for name in want[i]:
            assert torch.equal(out[name], want[i][name]), (i, name)
            assert torch.equal(eager[name], want[(i + 1) % 3][name]), (i, name)
