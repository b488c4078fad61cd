"""EdgeGraphTransformerLayer and a training step of a whole node classifier (layers, a
last norm, the loss), forward and backward, against the same formula in 64 bits."""
from __future__ import annotations

import pytest
import torch

from _edge_reference import adjacency, forward
from conftest import random_csr

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]


def layer_in_64(layer, p, x, adj, positions):
    F = torch.nn.functional
    n, H, C = x.shape[0], layer.heads, x.shape[1]
    norm = lambda t, name: F.layer_norm(t, (C,), p[name + ".weight"], p[name + ".bias"], 1e-5)
    dense = lambda t, name: F.linear(t, p[name + ".weight"], p[name + ".bias"])
    q, k, v = dense(norm(x, "norm1"), "qkv").view(n, 3, H, 64).unbind(1)
    o = forward(q, k, v, p.get("slopes"), positions, adj, layer.scale, layer.cap)
    y = dense(o.reshape(n, H * 64), "proj") + x
    if layer.up is None:
        return y
    return dense(F.gelu(dense(norm(y, "norm2"), "up")), "down") + y


def make(dtype, n=500, dim=96, H=2, **more):
    from fused3s_amd.torch_ops import EdgeGraphTransformerLayer, TorchGraph
    rp, ci = random_csr(n, 6, 4)
    graph = TorchGraph(rp, ci, heads=H)
    torch.manual_seed(2)
    layer = EdgeGraphTransformerLayer(dim, heads=H, **more).cuda().to(dtype)
    gen = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        for name, t in layer.named_parameters():
            if "norm" in name:
                t.add_(0.2 * torch.randn(t.shape, generator=gen, device="cuda"))
    x = torch.randn(n, dim, generator=gen, device="cuda").to(dtype)
    dy = torch.randn(n, dim, generator=gen, device="cuda").to(dtype)
    positions = 2 * torch.randn(n, 3, generator=gen, device="cuda") if more.get("distance") else None
    return layer, graph, x, dy, positions, adjacency(n, rp, ci).cuda()


def leaves_of(*modules):
    return {f"{i}.{name}": t for i, m in enumerate(modules) for name, t in m.named_parameters()}


def in_64(leaves):
    return {name: t.detach().double().requires_grad_() for name, t in leaves.items()}


def part(p, i):
    return {name[len(str(i)) + 1:]: t for name, t in p.items() if name.startswith(f"{i}.")}


@pytest.mark.parametrize("more", [dict(ffn_dim=200, cap=4.0, distance=True), dict(ffn_dim=128),
                                  dict(cap=2.0), dict(distance=True)])
@pytest.mark.parametrize("dtype", HALF)
def test_step(gpu, dtype, more):
    layer, graph, x, dy, positions, adj = make(dtype, **more)
    leaf = x.detach().requires_grad_()
    leaves = {**leaves_of(layer), "x": leaf}
    y = layer(leaf, graph, positions)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    p = in_64(leaves)
    want = layer_in_64(layer, part(p, 0), p["x"], adj, positions)
    exact = dict(zip(p, torch.autograd.grad(want, list(p.values()), dy.double())))
    # Up to 14 tensors between an input and a gradient are rounded, each by half a step
    # of its values at most, and pass on by a gain of 2 at most: 28 half-steps.  (The
    # slopes: a difference of sums over a row's edges, 4 times more.)
    bound = 28 * torch.finfo(dtype).eps / 2
    assert (y.double() - want).norm() <= bound * want.norm()
    for name, g in grads.items():
        times = 4 if "slopes" in name else 1
        assert (g.double() - exact[name]).norm() <= times * bound * exact[name].norm(), name
    with torch.no_grad():
        assert torch.equal(layer(x, graph, positions), y)


@pytest.mark.parametrize("dtype", HALF)
def test_training_a_classifier(gpu, dtype):
    """Two layers, a last norm, the loss of 1,000 classes: the loss and every gradient."""
    from fused3s_amd.torch_ops import layer_norm, linear_cross_entropy
    more = dict(ffn_dim=128, cap=4.0, distance=True)
    a, graph, x, _, positions, adj = make(dtype, **more)
    b = make(dtype, **more)[0]
    gen = torch.Generator(device="cuda").manual_seed(5)
    head = torch.nn.Linear(96, 1000).cuda().to(dtype)
    last = torch.nn.LayerNorm(96).cuda().to(dtype)
    target = torch.randint(1000, (500,), generator=gen, device="cuda")
    target[::5] = -100
    leaves = leaves_of(a, b, head, last)
    scale = torch.tensor(1024.0, device="cuda")   # (of the loss: binary16's gradients)
    h = layer_norm(b(a(x, graph, positions), graph, positions), last.weight, last.bias)
    loss = linear_cross_entropy(h, head.weight, target, head.bias)
    grads = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()), scale)))
    p = in_64(leaves)
    y = layer_in_64(b, part(p, 1), layer_in_64(a, part(p, 0), x.double(), adj, positions), adj,
                    positions)
    F = torch.nn.functional
    y = F.layer_norm(y, (96,), p["3.weight"], p["3.bias"], 1e-5)
    want = F.cross_entropy(F.linear(y, p["2.weight"], p["2.bias"]), target)
    exact = dict(zip(p, torch.autograd.grad(want, list(p.values()), scale.double())))
    # 14 tensors a layer, one for the norm, one for the logits' gradient: 30 of them each
    # way, a gain of 2 each: 120 half-steps
    bound = 120 * torch.finfo(dtype).eps / 2
    assert abs(float(loss.detach()) - float(want.detach())) <= bound * float(want.detach())
    for name, g in grads.items():
        times = 4 if "slopes" in name else 1
        assert (g.double() - exact[name]).norm() <= times * bound * exact[name].norm(), name


def test_captured_step(gpu):
    """A captured step of the layer and the loss, replayed with new inputs between eager
    work, each replay against the eager result."""
    from fused3s_amd.torch_ops import linear_cross_entropy
    layer, graph, x, _, positions, _ = make(torch.bfloat16, ffn_dim=64, cap=3.0, distance=True)
    graph.prepare_backward()
    gen = torch.Generator(device="cuda").manual_seed(9)
    w = (0.1 * torch.randn(40, 96, generator=gen, device="cuda")).bfloat16()
    target = torch.randint(40, (500,), generator=gen, device="cuda")

    def step(x, leaves):
        loss = linear_cross_entropy(layer(x, graph, positions), leaves[0], target)
        return loss.detach(), torch.autograd.grad(loss, leaves)

    captured = [t.detach().clone().requires_grad_() for t in (w,)]
    static = x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(static, captured)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss, grads = step(static, captured)
    for i in range(3):
        new = torch.randn(500, 96, generator=gen, device="cuda").bfloat16()
        static.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        eager_loss, eager = step(new, [w.detach().requires_grad_()])
        assert torch.equal(loss, eager_loss) and torch.equal(grads[0], eager[0])


def test_watched_and_hooked_modules_are_torchs(gpu):
    layer, graph, x, _, _, _ = make(torch.bfloat16, ffn_dim=64)
    with torch.no_grad():
        plain = layer(x, graph)
        calls = []
        handle = layer.norm1.register_forward_hook(lambda m, i, o: calls.append(o.shape))
        hooked = layer(x, graph)
        handle.remove()
        assert calls == [x.shape]
        # (torch's norm rounds as this one does, by half a step of each value at most)
        bound = 28 * torch.finfo(torch.bfloat16).eps / 2
        assert (hooked.double() - plain.double()).norm() <= bound * plain.double().norm()
        layer.norm1.double()
        layer.norm1.to(torch.bfloat16)
        assert torch.equal(layer(x, graph), plain)


def test_float32_module(gpu):
    layer, graph, x, _, positions, adj = make(torch.float32, ffn_dim=64, distance=True)
    with torch.no_grad():
        y = layer(x, graph, positions)
        p = {name: t.double() for name, t in layer.named_parameters()}
        want = layer_in_64(layer, p, x.double(), adj, positions)
    assert y.dtype is torch.float32
    # (the attention's operands and result in binary16)
    assert (y.double() - want).norm() <= 8 * 2.0 ** -11 * want.norm()


def test_refusals(gpu):
    from fused3s_amd.torch_ops import EdgeGraphTransformerLayer, TorchGraph
    layer, graph, x, _, positions, _ = make(torch.bfloat16, distance=True)
    with pytest.raises(ValueError, match="distance"):
        layer(x, graph)
    with pytest.raises(ValueError, match="distance"):
        make(torch.bfloat16)[0](x, graph, positions)
    rp, ci = random_csr(500, 6, 4)
    with pytest.raises(ValueError, match="head count"):
        layer(x, TorchGraph(rp, ci, heads=1), positions)
    with pytest.raises(ValueError, match="activation"):
        EdgeGraphTransformerLayer(64, activation="tanh")
