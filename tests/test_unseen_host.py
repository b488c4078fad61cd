"""The operators that call kernels on data pointers, where torch would not see the
call: under tracing, functorch's transforms and forward-mode differentiation they
refuse, on any host, before they look at a device; elsewhere they do not."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

N, H = 6, 2


def calls():
    """name -> (the call of one tensor, that tensor); past the refusal each raises
    ValueError here, where no tensor is on a device."""
    from fused3s_amd.torch_ops import TorchGraph, linear
    graph = TorchGraph.__new__(TorchGraph)   # (its own __init__ needs a device)
    graph.n, graph.heads, graph.masked, graph.device = N, H, False, 0
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)
    x, w, q, q64, lam = half(N, 8), half(4, 8), half(N, H, 128), half(N, H, 64), torch.zeros(H)
    return {
        "linear": (lambda t: linear(t, w), x),
        "linear weight": (lambda t: linear(x, t), w),
        "linear bias": (lambda t: linear(x, w, t), half(4)),
        "linear residual": (lambda t: linear(x, w, None, "gelu", t), half(N, 4)),
        "diff_attention": (lambda t: graph.diff_attention(t, q, q, lam), q),
        "diff_attention v": (lambda t: graph.diff_attention(q, q, t, lam), q),
        "diff_attention lam": (lambda t: graph.diff_attention(q, q, q, t), lam),
        "diff_attention_packed": (lambda t: graph.diff_attention_packed(t, lam), half(N, 3 * H * 128)),
        "attention": (lambda t: graph.attention(q64, t, q64), q64),
        "attention_packed": (lambda t: graph.attention_packed(t), half(N, 3 * H * 64)),
    }


NAMES = list(calls())


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    call, x = calls()[name]
    for grad in (torch.enable_grad, torch.no_grad):
        with grad(), forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
            with pytest.raises(ValueError):   # (no tangent: no business of the refusal)
                call(x)


@pytest.mark.parametrize("name", NAMES)
def test_tracing_is_refused(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    call, x = calls()[name]
    refused = pytest.raises(RuntimeError, match="cannot be traced")
    for how in ({}, {"tracing_mode": "fake"}, {"tracing_mode": "symbolic"}, {"pre_dispatch": True}):
        with refused:
            make_fx(call, **how)(x)
    with refused:
        torch.jit.trace(call, x, check_trace=False)
    with refused, FakeTensorMode(allow_non_fake_inputs=True):
        call(x)
    for transform in (torch.func.functionalize, torch.func.grad):
        with refused:
            transform(lambda t: call(t).float().sum())(x)
    with refused:
        torch.func.vmap(call)(x[None])
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(call, (x,), (x,))
    with refused:
        torch.export.export(Module(call), (x,), strict=False)


class Module(torch.nn.Module):
    def __init__(self, call):
        super().__init__()
        self.call = call

    def forward(self, x):
        return self.call(x)


@pytest.mark.parametrize("name", NAMES)
def test_onlookers_are_not(name):
    """A mode that counts, a function mode, an inference mode or autocast change
    nothing: the call goes on to its own checks."""
    from torch.overrides import BaseTorchFunctionMode
    from torch.utils.flop_counter import FlopCounterMode
    call, x = calls()[name]
    for context in (FlopCounterMode(display=False), BaseTorchFunctionMode(),
                    torch.inference_mode(), torch.autocast("cpu", dtype=torch.bfloat16),
                    torch.device("cpu")):
        with context, pytest.raises(ValueError):
            call(x)
    # a transform of something else
    with pytest.raises(ValueError):
        torch.func.vmap(lambda t: call(x) + t)(torch.zeros(3))


def test_compiled_calls():
    """torch.compile: a call of forward mode is refused there too, in whichever
    order the compilations come; others reach the call's own checks."""
    call, x = calls()["linear"]
    f = torch.compile(lambda t: call(t) + 1, backend="eager")
    for _ in range(2):
        with pytest.raises(ValueError):
            f(x)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))


class Wrapper(torch.Tensor):
    """A tensor that stands for another one and has no memory of its own."""

    @staticmethod
    def __new__(cls, inner):
        t = torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype,
                                                device=inner.device)
        t.inner = inner
        return t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        inner = lambda t: t.inner if isinstance(t, Wrapper) else t
        return func(*map(inner, args), **(kwargs or {}))


class Named(torch.Tensor):
    """A subclass that is its own memory."""


@pytest.mark.parametrize("name", NAMES)
def test_wrappers_are_refused(name):
    """(A wrapper's data pointer is NULL: as bias or residual it would be left out.)"""
    call, x = calls()[name]
    with pytest.raises(TypeError, match="takes no Wrapper"):
        call(Wrapper(x))
    with pytest.raises(ValueError):
        call(x.as_subclass(Named))
