"""Sizes at which linear()'s products take the tiles of large cases, several of them
per workgroup, with ends inside tiles; and the query that says so."""
from __future__ import annotations

import ctypes as C
from collections import namedtuple

Tiling = namedtuple("Tiling", "kernel tile splits tiles workgroups pieces")
FORWARD, SLOPE, DX, DW = range(4)
FEW_ROWS, W_IN_LDS, TILES = range(3)

WIDE = [(12_300, 1000, 4104), (12_300, 1000, 4101), (2100, 8200, 2056), (1030, 8200, 8200),
        (4100, 2056, 8200), (8200, 1024, 4101), (17_000, 1544, 2056), (40_000, 264, 136),
        (30_011, 65, 264), (30_000, 64, 265), (70_001, 266, 520), (70_001, 264, 520)]


def tiling(n, K, M, act, bias, product) -> Tiling:
    """f3s_linear_tiling."""
    from fused3s_amd import _lib
    o = C.c_int32(), C.c_int32(), C.c_int32(), C.c_int64(), C.c_int64(), C.c_int32()
    assert _lib.hip().f3s_linear_tiling(n, K, M, act, bias, product, *map(C.byref, o)) == 0
    return Tiling(*(x.value for x in o))
