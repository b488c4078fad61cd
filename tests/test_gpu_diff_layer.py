"""DiffGraphTransformerLayer: the projections, differential attention and the
feed-forward part together, forward and backward, against the same module's
formula in 64 bits."""
from __future__ import annotations

import pytest
import torch

from _diff_reference import adjacency, forward
from conftest import random_csr

pytestmark = pytest.mark.gpu


def reference(layer, x, adj):
    """The layer in 64 bits; returns y and the leaves."""
    p = {k: t.detach().double().requires_grad_() for k, t in layer.named_parameters()}
    x = x.detach().double().requires_grad_()
    F = torch.nn.functional
    n, H = x.shape[0], layer.heads
    q, k, v = F.linear(x, p["qkv.weight"], p["qkv.bias"]).view(n, 3, H, 128).unbind(1)
    lam = (torch.exp((p["lambda_q1"] * p["lambda_k1"]).sum(-1))
           - torch.exp((p["lambda_q2"] * p["lambda_k2"]).sum(-1)) + layer.lambda_init)
    o = forward(q, k, v, lam, adj, layer.scale)
    o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + layer.eps)
    o = o * p["norm"] * (1 - layer.lambda_init)
    y = F.linear(o.reshape(n, H * 128), p["proj.weight"], p["proj.bias"]) + x
    z = F.gelu(F.linear(y, p["up.weight"], p["up.bias"]))
    return F.linear(z, p["down.weight"], p["down.bias"]) + y, {**p, "x": x}


def make(dtype, n=500, dim=96, H=2):
    from fused3s_amd.torch_ops import DiffGraphTransformerLayer, TorchGraph
    rp, ci = random_csr(n, 6, 4)
    graph = TorchGraph(rp, ci, heads=H)
    torch.manual_seed(2)
    layer = DiffGraphTransformerLayer(dim, heads=H, ffn_dim=200).cuda().to(dtype)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, dim, generator=gen, device="cuda").to(dtype)
    dy = torch.randn(n, dim, generator=gen, device="cuda").to(dtype)
    return layer, graph, x, dy, adjacency(n, rp, ci).cuda()


def step(layer, graph, x, dy):
    x = x.detach().clone().requires_grad_()
    leaves = dict(layer.named_parameters(), x=x)
    y = layer(x, graph)
    return y.detach(), dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_step(gpu, dtype):
    layer, graph, x, dy, adj = make(dtype)
    y, grads = step(layer, graph, x, dy)
    want, leaves = reference(layer, x, adj)
    exact = dict(zip(leaves, torch.autograd.grad(want, list(leaves.values()), dy.double())))
    # Up to 12 tensors between an input and a gradient are rounded, each by half a
    # step of its values at most, and pass on by a gain of 2 at most: 24 half-steps.
    # (lambda's vectors: their products of 64 terms near 0.1 cancel, 4 times more.)
    bound = 24 * torch.finfo(dtype).eps / 2
    assert (y.double() - want).norm() <= bound * want.norm()
    for name, g in grads.items():
        assert g.dtype == leaves[name].dtype or g.dtype == dtype
        times = 4 if name.startswith("lambda") else 1
        assert (g.double() - exact[name]).norm() <= times * bound * exact[name].norm(), name


def test_no_grad_and_training_agree(gpu):
    layer, graph, x, dy, _ = make(torch.bfloat16)
    y, _ = step(layer, graph, x, dy)
    with torch.no_grad():
        assert torch.equal(layer(x, graph), y)


def test_watched_and_hooked_products_are_torchs(gpu):
    """A hook on a projection or a mode around the layer sees torch's own
    products; the results differ by roundings (the activation's and the residual's
    inputs are rounded too)."""
    from torch.utils.flop_counter import FlopCounterMode
    layer, graph, x, dy, _ = make(torch.float16)
    want, _ = step(layer, graph, x, dy)
    seen = []
    hook = layer.up.register_forward_hook(lambda *a: seen.append(1))
    y, _ = step(layer, graph, x, dy)
    hook.remove()
    assert seen and (y - want).abs().max() <= 2.0 ** -8 * want.abs().max()
    with torch.no_grad(), FlopCounterMode(display=False) as counter:
        layer(x, graph)
    n, dim = x.shape
    assert counter.get_total_flops() == 2 * n * (dim * 768 + 256 * dim + 2 * dim * 200)


def test_float32_module(gpu):
    layer, graph, x, dy, adj = make(torch.float32)
    y, grads = step(layer, graph, x, dy)
    want, _ = reference(layer, x, adj)
    assert y.dtype == torch.float32
    assert (y.double() - want).norm() <= 12 * 2.0 ** -11 * want.norm()   # (attention in float16)


def test_captured_inference(gpu):
    layer, graph, x, _, _ = make(torch.bfloat16)
    with torch.no_grad():
        layer(x, graph)
        torch.cuda.synchronize()
        static = x.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(static, graph)
        for seed in range(3):
            torch.manual_seed(seed)
            fresh = torch.randn_like(x)
            static.copy_(fresh)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, layer(fresh, graph))


def test_refusals(gpu):
    from fused3s_amd.torch_ops import DiffGraphTransformerLayer
    layer, _, x, _, _ = make(torch.float16)
    _, other, *_ = make(torch.float16, H=3)
    with pytest.raises(ValueError, match="head count"):
        layer(x, other)
    with pytest.raises(ValueError, match="residual"):
        DiffGraphTransformerLayer(64, out_dim=32)
    with pytest.raises(ValueError, match="activation"):
        DiffGraphTransformerLayer(64, activation="tanh")
    assert DiffGraphTransformerLayer(64, out_dim=32, residual=False).proj.out_features == 32
