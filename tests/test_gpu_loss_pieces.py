"""The loss of a classifier of more than 256 inputs, whose logits' gradient goes through
memory in pieces: classes and rows past the first piece, and the last, smaller one."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from _loss_reference import Reference
from test_gpu_loss import check, inputs, same, step

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]


def workspace(n, K, V, backward):
    from fused3s_amd import _lib
    need = C.c_int64()
    assert _lib.hip().f3s_cross_entropy_workspace(n, K, V, backward, C.byref(need)) == 0
    return need.value


@pytest.mark.parametrize("bias", [True, False], ids=["bias", ""])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,K,V", [(20_000, 264, 16_001), (20_000, 301, 16_001), (70_001, 272, 9000)])
def test_pieces_of_the_classes(gpu, n, K, V, dtype, bias):
    """Two pieces and more, the last one smaller and ragged; each gradient alone."""
    from fused3s_amd.torch_ops import linear_cross_entropy
    copies = 4 * (n + V) * (K + 7) if K % 8 else 0
    assert workspace(n, K, V, 1) - copies < 2 * n * V   # (all of the logits' gradient)
    x, w, b, t, dloss = inputs(n, K, V, dtype, 4, bias)
    got = step(x, w, b, t, dloss, "mean")
    check(got, x, w, b, t, dloss, "mean")
    same(got, step(x, w, b, t, dloss, "mean"))
    for i, name in ((0, "dx"), (1, "dw"), (2, "db")):
        leaves = [x, w, b]
        if leaves[i] is None:
            continue
        leaves[i] = leaves[i].detach().requires_grad_()
        g, = torch.autograd.grad(linear_cross_entropy(leaves[0], leaves[1], t, leaves[2]), [leaves[i]],
                                 dloss)
        assert torch.equal(g, got[name]), name


@pytest.mark.parametrize("n,K,V", [(70_000, 264, 17_000), (70_000, 257, 17_000), (900_000, 264, 1000)])
def test_pieces_of_the_rows(gpu, n, K, V):
    """More blocks than a forward pass holds at a time."""
    from fused3s_amd.torch_ops import linear_cross_entropy
    copies = 2 * (n + V) * (K + 7) if K % 8 else 0
    assert workspace(n, K, V, 0) - copies - 4 * n - 16 * n // 4 < 8 * n * (V // 32 + 8)
    x, w, b, t, _ = inputs(n, K, V, torch.bfloat16, 5, reduction="none")
    with torch.no_grad():
        loss = linear_cross_entropy(x, w, t, b, reduction="none")
        total = linear_cross_entropy(x, w, t, b, reduction="sum")
    for r0 in range(0, n, n // 7):
        at = slice(r0, r0 + n // 7)
        Reference(x[at], w, b, t[at], "none").check("loss", loss[at])
    assert abs(float(loss.double().sum()) - float(total)) <= 2.0 ** -23 * float(total)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,K,V", [(300_000, 264, 1500), (300_001, 301, 3001), (262_145, 320, 70)])
def test_blocks_of_the_rows(gpu, n, K, V, dtype):
    """More rows than the logits' gradient is taken of at a time, one piece of the classes
    and several; each gradient alone."""
    from fused3s_amd.torch_ops import linear_cross_entropy
    x, w, b, t, dloss = inputs(n, K, V, dtype, 6, ignored=0.5)
    got = step(x, w, b, t, dloss, "mean")
    check(got, x, w, b, t, dloss, "mean")
    same(got, step(x, w, b, t, dloss, "mean"))
    for i, name in ((0, "dx"), (1, "dw"), (2, "db")):
        leaves = [x, w, b]
        leaves[i] = leaves[i].detach().requires_grad_()
        g, = torch.autograd.grad(linear_cross_entropy(leaves[0], leaves[1], t, leaves[2]), [leaves[i]],
                                 dloss)
        assert torch.equal(g, got[name]), name
