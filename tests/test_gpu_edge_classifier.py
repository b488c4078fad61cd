"""A training step of a node classifier (two layers, a last norm, the loss), every gradient
as near to 64 bits as the same network of torch's operations in the same type, or within
three times its error."""
from __future__ import annotations

import pytest
import torch

from _edge_reference import forward
from test_gpu_edge_layer import HALF, in_64, layer_in_64, leaves_of, make, part

pytestmark = pytest.mark.gpu
F = torch.nn.functional


def layer_in_torch(layer, p, x, adj, positions):
    """The layer of 16-bit tensors: each operation's result rounded, attention's inside in
    64 bits."""
    n, H, C = x.shape[0], layer.heads, x.shape[1]
    norm = lambda t, name: F.layer_norm(t, (C,), p[name + ".weight"], p[name + ".bias"], 1e-5)
    dense = lambda t, name: F.linear(t, p[name + ".weight"], p[name + ".bias"])
    q, k, v = (t.double() for t in dense(norm(x, "norm1"), "qkv").view(n, 3, H, 64).unbind(1))
    # (slopes are float32 in the layer)
    o = forward(q, k, v, p["slopes"].float(), positions, adj, layer.scale, layer.cap).to(x.dtype)
    y = dense(o.reshape(n, H * 64), "proj") + x
    return dense(F.gelu(dense(norm(y, "norm2"), "up")), "down") + y


@pytest.mark.parametrize("dtype", HALF)
def test_as_near_as_torch(gpu, dtype):
    from fused3s_amd.torch_ops import layer_norm, linear_cross_entropy
    more = dict(ffn_dim=128, cap=4.0, distance=True)
    a, graph, x, _, positions, adj = make(dtype, **more)
    b = make(dtype, **more)[0]
    gen = torch.Generator(device="cuda").manual_seed(5)
    head = torch.nn.Linear(96, 1000).cuda().to(dtype)
    last = torch.nn.LayerNorm(96).cuda().to(dtype)
    target = torch.randint(1000, (500,), generator=gen, device="cuda")
    target[::5] = -100
    scale = torch.tensor(1024.0, device="cuda")   # (of the loss: binary16's gradients)
    leaves = leaves_of(a, b, head, last)

    def grads_of(loss, p):
        return loss.detach(), dict(zip(p, torch.autograd.grad(loss, list(p.values()),
                                                              scale.to(loss.dtype))))

    h = layer_norm(b(a(x, graph, positions), graph, positions), last.weight, last.bias)
    loss, grads = grads_of(linear_cross_entropy(h, head.weight, target, head.bias), leaves)

    def plain(p, layer, wide):
        y = layer(b, part(p, 1), layer(a, part(p, 0), wide(x), adj, positions), adj, positions)
        y = F.layer_norm(y, (96,), p["3.weight"], p["3.bias"], 1e-5)
        # (logits are not rounded)
        up = (lambda t: t) if y.dtype == torch.float64 else torch.Tensor.float
        return F.cross_entropy(F.linear(up(y), up(p["2.weight"]), up(p["2.bias"])), target)

    p = in_64(leaves)
    want, exact = grads_of(plain(p, layer_in_64, torch.Tensor.double), p)
    p = {name: t.detach().clone().requires_grad_() for name, t in leaves.items()}
    theirs, torchs = grads_of(plain(p, layer_in_torch, lambda t: t), p)
    assert len(grads) == len(leaves) and any("slopes" in name for name in grads)
    # the loss: within three roundings of its last hidden values, a step of the type each
    eps = torch.finfo(dtype).eps
    assert abs(float(loss) - float(want)) <= 3 * eps * float(want)
    for name, g in grads.items():
        size = exact[name].norm()
        ours, other = ((t[name].double() - exact[name]).norm() / size for t in (grads, torchs))
        bound = 3 * other + eps   # (and a rounding of either)
        assert float(bound) < 0.1, (name, float(bound))   # (a term left out would be seen)
        assert float(ours) <= float(bound), (name, float(ours), float(other))
