"""Edge attention, the layer norm and the classifier's loss where torch would not see their
kernels' calls: the refusals of test_unseen_host, each tensor of theirs in turn."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import test_unseen_host as host

N, H = host.N, host.H


def calls():
    from fused3s_amd.torch_ops import TorchGraph, layer_norm, linear_cross_entropy
    graph = TorchGraph.__new__(TorchGraph)   # (its own __init__ needs a device)
    graph.n, graph.heads, graph.masked, graph.device = N, H, False, 0
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)
    q, qkv, pos, slopes = half(N, H, 64), half(N, 3 * H * 64), torch.zeros(N, 2), torch.zeros(H)
    x, w, b, classes = half(N, 8), half(5, 8), half(5), torch.zeros(N, dtype=torch.int64)
    edge = lambda *qkv, **more: graph.edge_attention(*qkv, 0.125, 30.0, **more)
    return {
        "edge_attention": (lambda t: edge(t, q, q), q),
        "edge_attention k": (lambda t: edge(q, t, q), q),
        "edge_attention v": (lambda t: edge(q, q, t), q),
        "edge_attention positions": (lambda t: edge(q, q, q, positions=t, slopes=slopes), pos),
        "edge_attention slopes": (lambda t: edge(q, q, q, positions=pos, slopes=t), slopes),
        "edge_attention_packed": (lambda t: graph.edge_attention_packed(t), qkv),
        "edge_attention_packed slopes": (
            lambda t: graph.edge_attention_packed(qkv, positions=pos, slopes=t), slopes),
        "layer_norm": (lambda t: layer_norm(t), x),
        "layer_norm weight": (lambda t: layer_norm(x, t), half(8)),
        "layer_norm bias": (lambda t: layer_norm(x, None, t), half(8)),
        "linear_cross_entropy": (lambda t: linear_cross_entropy(t, w, classes), x),
        "linear_cross_entropy weight": (lambda t: linear_cross_entropy(x, t, classes), w),
        "linear_cross_entropy bias": (lambda t: linear_cross_entropy(x, w, classes, t), b),
    }


NAMES = list(calls())


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("test", [host.test_forward_mode_is_refused, host.test_tracing_is_refused,
                                  host.test_onlookers_are_not])
def test_unseen(monkeypatch, test, name):
    monkeypatch.setattr(host, "calls", calls)
    test(name)


@pytest.mark.parametrize("name", ["linear_cross_entropy", "layer_norm", "edge_attention"])
def test_compiled_calls(monkeypatch, name):
    call = calls()[name]
    monkeypatch.setattr(host, "calls", lambda: {"linear": call})
    host.test_compiled_calls()
