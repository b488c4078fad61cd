"""The workspace of the loss's backward pass, at most what its documentation says, over rows
and classes of every size."""
from __future__ import annotations

import ctypes as C

import pytest

from fused3s_amd import _lib

MIB = 1 << 20


def workspace(n, K, V, backward):
    need = C.c_int64()
    assert _lib.hip().f3s_cross_entropy_workspace(n, K, V, backward, C.byref(need)) == 0
    return need.value


@pytest.mark.parametrize("n", [1, 64, 1000, 16_384, 70_000, 262_144, 262_145, 500_000, 1_000_000, 8_200_001,
                               54_000_000])
@pytest.mark.parametrize("V", [65, 1000, 4000, 10_000, 100_003, 1_000_000])
def test_more_than_256_inputs(n, V):
    """512 MB of the logits' gradient (and a sixteenth of that, its column sums), dx of a
    block of rows in float32, past 262,144 rows dW in float32; splits of either (256 MB)."""
    for K in (264, 400, 512, 1024):
        rows = 4 * min(n, 262_144) * K + (4 * V * (K + 1) if n > 262_144 else 0)
        assert workspace(n, K, V, 1) <= 512 * MIB * 17 // 16 + rows + 256 * MIB + 8 * n, (n, K, V)
    # (what is copied first where rows are no whole pieces: x, W and their gradients)
    for K, Kp in ((257, 264), (301, 304)):
        copies = 4 * (n + V) * Kp
        assert workspace(n, K, V, 1) <= workspace(n, Kp, V, 1) + copies + 512 * MIB


@pytest.mark.parametrize("n", [1, 64, 1000, 16_384, 200_003, 500_000, 1_000_000, 8_200_001, 54_000_000])
@pytest.mark.parametrize("V", [2, 64, 65, 1000, 10_000, 100_003, 1_000_000, 54_000_000])
def test_up_to_256_inputs(n, V):
    """512 MB of the gradients' slices; db's, of up to 4,096 shares of the rows of few
    classes and few of many."""
    for K in (8, 64, 128, 136, 256):
        assert workspace(n, K, V, 1) <= 512 * MIB + 8 * n + 64 * MIB + 4 * 16 * V, (n, K, V)
        # (forward: 8 bytes a row and share of the classes)
        assert workspace(n, K, V, 0) <= 80 * n + 64 * MIB, (n, K, V)
