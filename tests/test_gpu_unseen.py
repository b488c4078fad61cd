"""On a device: what torch cannot see is refused by the layers too, and what only
looks on, or compiles around the calls, gets their results."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from conftest import random_csr

pytestmark = pytest.mark.gpu


def layers():
    from fused3s_amd.torch_ops import (DiffGraphTransformerLayer, GraphTransformerLayer,
                                       TorchGraph)
    rp, ci = random_csr(300, 5, 2)
    torch.manual_seed(0)
    x = torch.randn(300, 64, device="cuda").half()
    graph = TorchGraph(rp, ci, heads=2).prepare_backward()
    for kind, more in ((GraphTransformerLayer, {}), (DiffGraphTransformerLayer, {"ffn_dim": 128})):
        yield kind(64, heads=2, **more).cuda().half(), graph, x


def test_layers_refuse(gpu):
    from torch.fx.experimental.proxy_tensor import make_fx
    for layer, graph, x in layers():
        layer.requires_grad_(False)
        for grad in (torch.no_grad, torch.enable_grad):
            with grad():
                with forward_ad.dual_level():
                    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                        layer(forward_ad.make_dual(x, torch.ones_like(x)), graph)
                with pytest.raises(RuntimeError, match="cannot be traced"):
                    make_fx(lambda t: layer(t, graph))(x)
                with pytest.raises(RuntimeError, match="cannot be traced"):
                    torch.jit.trace(lambda t: layer(t, graph), x, check_trace=False)


def test_onlookers_see_the_results(gpu):
    from torch.utils.flop_counter import FlopCounterMode

    from fused3s_amd.torch_ops import linear
    for layer, graph, x in layers():
        want = layer(x, graph)
        bound = 2.0 ** -8 * want.abs().max()   # (projections by torch, rounded between)
        with FlopCounterMode(display=False):
            assert (layer(x, graph) - want).abs().max() <= bound
    compiled = torch.compile(layer, backend="eager")   # (the trainable one)
    assert (compiled(x, graph) - want).abs().max() <= bound
    w = torch.randn(40, 64, device="cuda").half().requires_grad_()
    want = linear(x, w, None, "silu")
    assert torch.equal(torch.compile(lambda t: linear(t, w, None, "silu"), backend="eager")(x), want)
    with FlopCounterMode(display=False), torch.inference_mode():
        assert torch.equal(linear(x, w, None, "silu"), want)


class Counted(torch.Tensor):
    """A weight whose class sees its uses."""

    seen = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        Counted.seen.append(func)
        return super().__torch_function__(func, types, args, kwargs or {})


def test_weights_of_a_subclass_are_torchs(gpu):
    """A projection whose weight or bias is of a tensor subclass is torch's own, as
    the forward-only layer's is: the subclass sees the product."""
    for layer, graph, x in layers():
        with torch.no_grad():
            want = layer(x, graph).as_subclass(torch.Tensor)
            for name, p in list(layer.named_parameters()):
                module, _, leaf = name.rpartition(".")
                if leaf not in ("weight", "bias"):
                    continue
                owner = layer.get_submodule(module)
                setattr(owner, leaf, torch.nn.Parameter(p.detach().as_subclass(Counted),
                                                        requires_grad=False))
                Counted.seen.clear()
                y = layer(x, graph).as_subclass(torch.Tensor)
                assert torch.nn.functional.linear in Counted.seen, name
                assert (y - want).abs().max() <= 2.0 ** -8 * want.abs().max(), name
                setattr(owner, leaf, p)


def test_attention_follows_the_current_stream(gpu):
    """The forward-only passes run on torch's current stream: behind work that is
    still ahead of them there."""
    for layer, graph, x in layers():
        q = torch.randn(300, 2, 64, device="cuda").half()
        qkv = torch.randn(300, 384, device="cuda").half()
        want = graph.attention(q, q, q, 0.125), graph.attention_packed(qkv, 0.125)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            busy = torch.randn(4096, 4096, device="cuda")
            for _ in range(20):
                busy = busy @ busy * 1e-2
            late = q * 0, qkv * 0
            late[0].copy_(q)
            late[1].copy_(qkv)
            got = graph.attention(late[0], late[0], late[0], 0.125), graph.attention_packed(late[1], 0.125)
        side.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        break
