"""CPU test: the shapes that test_gpu_tiles.py runs on the GPU reach every tile that the entry
points of lsamp_blocks_api.cpp choose, for every operator (blocks_launches.cpp writes the
choices down)."""
from __future__ import annotations

import ctypes
from ctypes import c_void_p

import tile_shapes as S
from lsamp import _ffi
from test_blocks_plan import (GRAM, PARTIAL, POLY, PRODUCT, TILES, TYPES, UPDATE, Memory, lib,  # noqa: F401
                              run)

LARGE = {"64", "64x4", "128", "128x2", "192", "256"}


def _orth_tiles(lib, batch, rows, cols, fast):  # noqa: F811
    c = (ctypes.c_float * 3)(3.4445, -4.7750, 2.0315)
    mem = Memory()
    a = _ffi.OrthogonalizeArgs(batch=batch, rows=rows, cols=cols, in_dtype=_ffi.DTYPE_BF16,
                               out_dtype=_ffi.DTYPE_BF16, steps=1, eps=1e-7, scale=1.0, keep=1.0,
                               fast=fast, coefficients=ctypes.cast(c, c_void_p))
    a.x = mem.vector(batch * rows * cols, 2)
    a.out = mem.vector(batch * rows * cols, 2, True)
    a.x_stride = a.out_stride = cols
    a.x_batch_stride = a.out_batch_stride = rows * cols
    return {x.kind: TILES[x.tile] for x in run(lib, "lsamp_orthogonalize", a, mem) if x.tile >= 0}


def test_orthogonalize(lib):  # noqa: F811
    for fast in (0, 1):
        tiles = {}
        for batch, m, n in S.ORTH:
            for rows, cols in ((m, n), (n, m)):
                for kind, tile in _orth_tiles(lib, batch, rows, cols, fast).items():
                    # (B's product is the same one for both)
                    way = "" if kind == POLY else "tall" if rows > cols else "wide"
                    tiles.setdefault((kind, way), set()).add(tile)
        # (32x8: both operands' rows along the output; 192: symmetric products)
        assert tiles == {(GRAM, "wide"): LARGE | {"32x8"}, (GRAM, "tall"): LARGE,
                         (POLY, ""): LARGE | {"32x8"}, (UPDATE, "wide"): LARGE - {"192"},
                         (UPDATE, "tall"): (LARGE - {"192"}) | {"32x8"}}, (fast, tiles)


def test_linear_int8(lib):  # noqa: F811
    whole = {"64", "64x4", "128", "128x2", "256", "loose64", "loose64x4", "loose128"}
    for name, (dt, eb) in TYPES.items():
        tiles = {}
        for m, k, n, layout in S.INT8:
            odd = layout == "odd"
            mem = Memory()
            a = _ffi.LinearInt8Args(rows=m, in_features=k, out_features=n, dtype=dt, out_dtype=dt)

            def matrix(rows, cols, size, write=False):
                ld = cols + 3 * odd
                at = mem.vector(rows * ld + 1, size, write) + odd * size
                return at, ld
            a.x, a.x_stride = matrix(m, k, eb)
            a.weight, a.weight_stride = matrix(n, k, 1)
            a.weight_scale = mem.vector(n, 4)
            a.out, a.out_stride = matrix(m, n, eb, True)
            a.residual, a.residual_stride = matrix(m, n, eb)
            for x in run(lib, "lsamp_linear_int8", a, mem):
                if x.kind in (PARTIAL, PRODUCT):
                    tile = TILES[x.tile]
                    if tile.startswith("skinny"):
                        tile += "/16" if m <= 16 else "/32" if m <= 32 else "/64"
                    tiles.setdefault(x.kind, set()).add(tile)
        # (64 rows too long to be kept, of few and of many columns: test_gpu_blocks.py)
        some = {"skinny16/32", "skinny64/16", "skinny64/32"}
        assert tiles[PARTIAL] == whole, (name, tiles[PARTIAL] ^ whole)
        assert tiles[PRODUCT] == whole | some, (name, tiles[PRODUCT] ^ (whole | some))
