"""What linear()'s passes ask for as workspace, on any host."""
from __future__ import annotations

import ctypes as C

import pytest

pytest.importorskip("torch")

from fused3s_amd import _lib


def size(*a):
    need = C.c_int64()
    assert _lib.hip().f3s_linear_workspace(*a, C.byref(need)) == 0
    return need.value


@pytest.mark.parametrize("n,K,M", [(4096, 4096, 4096), (4096, 4096, 8192), (8192, 8192, 4096)])
def test_products_of_one_split_ask_for_no_sums(n, K, M):
    """dW of one split is written at once: the workspace is dz with its columns' sums
    (activation), or those of eight columns (db alone), not 4 M K bytes beside."""
    sums = 8 * M * ((n + 63) // 64) + 4 * 64 * M + 4 * M + 4 * 256
    assert size(n, K, M, 2, 1) <= 2 * n * M + sums
    assert size(n, K, M, 0, 1) <= 4 * M * 8 + 4 * M + 2 * 256
