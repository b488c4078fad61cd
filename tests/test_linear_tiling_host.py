"""Which tiles linear()'s products take, on any host: the sizes that the GPU tests run
cover every tile, with several of them per workgroup, in every product; a change of the
estimate that chooses them cannot drop one unseen."""
from __future__ import annotations

import ctypes as C

import pytest

pytest.importorskip("torch")

from _linear_sizes import DW, DX, FEW_ROWS, FORWARD, SLOPE, TILES, W_IN_LDS, WIDE, tiling
from fused3s_amd import _lib

RELU = 1


def taken(product, act, sizes=WIDE):
    """(tile, whether the contraction is split, pieces) of those sizes whose workgroups
    take several tiles each."""
    got = set()
    for size in sizes:
        t = tiling(*size, act, 1, product)
        if t.kernel == TILES and t.tiles > t.workgroups:
            got.add((t.tile, t.splits > 1, t.pieces))
    return got


@pytest.mark.parametrize("product", [FORWARD, SLOPE])
def test_forward_and_slope(product):
    assert taken(product, RELU) >= {(256, False, 2), (256, False, 1), (256, True, 2),
                                    (128, False, 2), (128, False, 1), (128, False, 0),
                                    (64, False, 2), (64, False, 1), (64, False, 0)}


def test_dx():
    assert taken(DX, RELU) >= {(256, False, 2), (256, True, 2), (128, False, 2), (128, False, 0),
                               (64, False, 2), (64, False, 0)}


def test_dw():
    assert taken(DW, RELU) >= {(256, False, 2), (256, True, 2), (128, False, 2), (128, True, 0)}
    # with db in the same product: no tiles of 256
    assert taken(DW, 0) >= {(128, False, 2), (128, True, 2), (128, True, 0)}
    assert all(tile < 256 for tile, *_ in taken(DW, 0))


def test_other_kernels():
    assert tiling(64, 1000, 4104, RELU, 1, FORWARD).kernel == FEW_ROWS
    assert tiling(65, 1000, 4104, RELU, 1, FORWARD).kernel == TILES
    assert tiling(49_152, 128, 512, RELU, 1, SLOPE).kernel == W_IN_LDS
    assert tiling(49_152, 512, 128, RELU, 1, DX).kernel == TILES
    assert tiling(98_304, 512, 128, RELU, 1, DX).kernel == W_IN_LDS


def test_refusals():
    call = lambda *a: _lib.hip().f3s_linear_tiling(*a, None, None, None, None, None, None)
    assert call(8, 8, 8, 0, 0, 0) == 0
    for bad in ((0, 8, 8, 0, 0, 0), (8, 8, 8, 0, 0, 4), (8, 8, 8, 0, 0, -1), (8, 0, 8, 0, 0, 0),
                (8, 8, 8, 5, 0, 0)):
        assert call(*bad) == 1
