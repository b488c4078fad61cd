"""f3s_plan_create_scheduled: the library's sequence from 513 windows on wherever masked
passes run no teams, past 1,024 window-heads; its passes against the oracle, and a step
of differential attention on it."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import _oracle as orc
from conftest import rng
from test_gpu_diff import check, inputs, step

pytestmark = pytest.mark.gpu

# windows, heads: both sides of 1,024 and 2,048 window-heads, few windows and many
SIZES = [(17, 64), (130, 8), (500, 3), (512, 4), (513, 2), (600, 2), (1030, 1), (2048, 1),
         (2049, 1)]


def slots(W):
    """Positions of a schedule of W windows: eight shares of W / 8, and a slot more per
    class of tile counts."""
    return 8 * (((W + 7) // 8 + 64 + 3) // 4 * 4)


def graph_of(W, seed, hubs=True):
    n, r = 16 * W - 7, rng(seed)
    keys = [r.integers(0, n, 3 * n) * np.int64(n) + r.integers(0, n, 3 * n)]
    for u in (3, n // 2, n - 1) if hubs else ():
        keys.append(u * np.int64(n) + np.arange(n))
    keys = np.unique(np.concatenate(keys))
    keys = keys[keys // n // 16 % 50 != 13]              # windows without an edge
    rp = np.searchsorted(keys // n, np.arange(n + 1)).astype(np.int32)
    return n, rp, (keys % n).astype(np.int32)


@pytest.mark.parametrize("W,H", SIZES)
def test_sequence(gpu, W, H):
    n, rp, ci = graph_of(W, W + H)
    bsf = gpu.convert_device(gpu.DeviceCSR(rp, ci))
    plan = gpu.Plan(bsf, H=H, scheduled=True)
    positions = 4 * W if W * H <= 1024 else slots(W) if W > 512 else W
    stats = plan.stats()
    # one item per position, and one more per further segment of a split window
    extra = stats["masked_slots"] - plan.num_split
    assert stats["masked_items"] == positions + extra
    plan.compile()
    r = rng(W)
    q, k, v = (r.standard_normal((n, H, 64)).astype(np.float16) for _ in range(3))
    dev = [gpu.DeviceArray.from_numpy(x.view(np.uint16)) for x in (q, k, v)]
    f = [x.astype(np.float32) for x in (q, k, v)]
    for masked in (True, False, True):
        out = gpu.DeviceArray((n, H, 64), np.float32)
        out.fill_bytes(0xff)   # NaN: a row that no item writes fails
        plan.forward(*dev, out, masked=masked, scale=0.125)
        gpu.synchronize()
        got = out.numpy()
        for h in (0, H - 1):
            g = [np.ascontiguousarray(x[:, h:h + 1]) for x in f]
            want = (orc.masked_attention(n, 64, 1, *g, rp, ci, 0.125) if masked else
                    orc.tile_dense_attention(n, 64, 1, *g, bsf.window_offsets.numpy(),
                                             bsf.block_col.numpy(), 0.125))
            assert np.abs(got[:, h:h + 1] - want).max() <= 2e-3, (masked, h)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("W,H", [(17, 64), (130, 8), (513, 2), (600, 2)])
def test_step(gpu, W, H, dtype):
    """A step on graphs of 1,025 to 2,048 window-heads: from 513 windows on the operator's
    plan and that of the reversed edges follow the schedule."""
    from fused3s_amd.torch_ops import TorchGraph
    n, rp, ci = graph_of(W, W, hubs=W < 200)
    graph = TorchGraph(rp, ci, heads=H).prepare_backward()
    for plan in (graph._diff_plan(), graph._reversed):
        assert plan.stats()["masked_items"] >= (slots(W) if W > 512 else W)
    q, k, v, lam, do = x = inputs(n, H, dtype, 5)
    got = step(graph, *x, 0.125)
    for h in (0, H // 2, H - 1) if H > 2 else range(H):
        part = [t[:, h:h + 1].contiguous() for t in (q, k, v)] + [lam[h:h + 1], do[:, h:h + 1].contiguous()]
        check({name: t[h:h + 1] if name == "dlam" else t[:, h:h + 1] for name, t in got.items()},
              *part, rp, ci, 0.125)
