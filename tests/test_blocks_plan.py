"""CPU tests of the launches that the entry points of lsamp_blocks_api.cpp make
(blocks_launches.cpp writes them down): every access ends inside a caller's matrix
or inside what an earlier launch wrote to the workspace, and every write inside an
output or the workspace."""
from __future__ import annotations

import ctypes
import os
import random
import subprocess
import tempfile
from ctypes import POINTER, byref, c_int32, c_int64, c_void_p

import pytest

from lsamp import _ffi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "mlx-swift-lm_amd", "csrc")
TYPES = {"f32": (_ffi.DTYPE_F32, 4), "bf16": (_ffi.DTYPE_BF16, 2), "f16": (_ffi.DTYPE_F16, 2)}
WORKSPACE = 1 << 44
(NORM, NORM_BACKWARD, QUANTIZE, PACK, PARTIAL, PRODUCT, RESIDENT, JOIN, START, GRAM, POLY,
 UPDATE) = range(12)
TILES = ("256", "128", "64", "128x2", "64x4", "loose128", "loose64", "loose64x4", "skinny64",
         "skinny16", "192", "32x8")


class Access(ctypes.Structure):
    _fields_ = [(f, c_int32) for f in "launch kind write tile".split()] + [("at", c_int64),
                                                                           ("bytes", c_int64)]


@pytest.fixture(scope="module")
def lib():
    with tempfile.TemporaryDirectory() as d:
        so = os.path.join(d, "blocks_launches.so")
        subprocess.run(
            ["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-w",
             "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + CSRC,
             os.path.join(CSRC, "lsamp_blocks_api.cpp"),
             os.path.join(REPO, "tests", "blocks_launches.cpp"), "-o", so], check=True)
        L = ctypes.CDLL(so)
    assert L.blocks_access_size() == ctypes.sizeof(Access)
    L.blocks_accesses.restype = c_int64
    for name, args in (("lsamp_layer_norm", _ffi.LayerNormArgs),
                       ("lsamp_layer_norm_backward", _ffi.LayerNormBackwardArgs),
                       ("lsamp_quantize_rows", _ffi.QuantizeRowsArgs),
                       ("lsamp_linear_int8", _ffi.LinearInt8Args),
                       ("lsamp_orthogonalize", _ffi.OrthogonalizeArgs)):
        getattr(L, name).argtypes = [c_void_p, POINTER(args), c_void_p]
        getattr(L, name).restype = c_int32
        if hasattr(args, "workspace") or hasattr(L, name + "_workspace"):
            getattr(L, name + "_workspace").argtypes = [POINTER(args)]
            getattr(L, name + "_workspace").restype = c_int64
    return L


class Memory:
    """Callers' arrays, far apart, with the bytes that they have."""

    def __init__(self):
        self.parts = []

    def matrix(self, rows, cols, eb, rng, write=False):
        ld = cols + rng.choice([0, 0, 8, 3])
        shift = rng.choice([0, 0, 1]) * eb
        at = (len(self.parts) + 1 << 50) + shift
        self.parts.append((at, ((rows - 1) * ld + cols) * eb, write))
        return at, ld

    def vector(self, n, eb, write=False):
        at = len(self.parts) + 1 << 50
        self.parts.append((at, n * eb, write))
        return at


def run(L, name, args, memory, sized=True):
    need = 0
    if sized:
        need = getattr(L, name + "_workspace")(byref(args))
        assert need >= 0
        args.workspace, args.workspace_bytes = WORKSPACE if need else None, need
    L.blocks_accesses(None, 0)
    assert getattr(L, name)(1, byref(args), None) == 0
    out = (Access * 4096)()
    n = L.blocks_accesses(out, 4096)
    assert n <= 4096
    written = []  # ranges of the workspace
    for a in out[:n]:
        end = a.at + a.bytes
        if WORKSPACE <= a.at < 1 << 50:
            assert end <= WORKSPACE + need, (a.kind, end - WORKSPACE, need)
            if a.write:
                written.append((a.at, end, a.launch))
            else:
                # (a buffer's reads begin anywhere in one that was written before)
                assert any(lo <= a.at and end <= hi and launch < a.launch
                           for lo, hi, launch in written), f"kind {a.kind} reads what is not written"
        else:
            assert any(at <= a.at and end <= at + size and (writable or not a.write)
                       for at, size, writable in memory.parts), f"kind {a.kind} outside a matrix"
    # buffers are apart: two writes of one call share all their bytes' first or none
    for lo, hi, _ in written:
        for lo2, hi2, _ in written:
            assert lo == lo2 or hi <= lo2 or hi2 <= lo, "buffers of the workspace overlap"
    return out[:n]


def test_norms(lib):
    rng = random.Random(1)
    for _ in range(200):
        dt, eb = TYPES[rng.choice(list(TYPES))]
        m, n = rng.choice([1, 3, 300, 513, 5000]), rng.choice([1, 77, 2048, 5000, 20000])
        mem = Memory()
        f = _ffi.LayerNormArgs(rows=m, cols=n, dtype=dt, eps=1e-5)
        f.x, f.x_stride = mem.matrix(m, n, eb, rng)
        f.out, f.out_stride = mem.matrix(m, n, eb, rng, True)
        f.weight, f.mean, f.rstd = mem.vector(n, eb), mem.vector(m, 4, True), mem.vector(m, 4, True)
        run(lib, "lsamp_layer_norm", f, mem, sized=False)
        b = _ffi.LayerNormBackwardArgs(rows=m, cols=n, dtype=dt, x=f.x, x_stride=f.x_stride,
                                       mean=f.mean, rstd=f.rstd, weight=f.weight)
        b.d_out, b.d_out_stride = mem.matrix(m, n, eb, rng, True)
        if rng.random() < 0.7:
            b.d_x, b.d_x_stride = mem.matrix(m, n, eb, rng, True)
            if rng.random() < 0.3:
                b.d_x, b.d_x_stride = b.d_out, b.d_out_stride
        if rng.random() < 0.7 or not b.d_x:
            b.d_weight = mem.vector(n, eb, True)
        run(lib, "lsamp_layer_norm_backward", b, mem)


def test_linear_int8(lib):
    rng = random.Random(2)
    kinds, tiles = set(), set()
    for _ in range(600):
        dt, eb = TYPES[rng.choice(list(TYPES))]
        m = rng.choice([1, 2, 4, 5, 16, 17, 64, 65, 300, 3000])
        k = rng.choice([1, 15, 16, 100, 128, 300, 2048, 2100, 9000])
        n = rng.choice([1, 70, 300, 4096, 40003, 70000])
        given = rng.random() < 0.4
        mem = Memory()
        a = _ffi.LinearInt8Args(rows=m, in_features=k, out_features=n, dtype=dt, out_dtype=dt)
        a.x, a.x_stride = mem.matrix(m, k, 1 if given else eb, rng)
        if given:
            a.x_scale = mem.vector(m, 4)
        a.weight, a.weight_stride = mem.matrix(n, k, 1, rng)
        a.weight_scale = mem.vector(n, 4)
        a.out, a.out_stride = mem.matrix(m, n, eb, rng, True)
        a.residual, a.residual_stride = mem.matrix(m, n, eb, rng)
        for x in run(lib, "lsamp_linear_int8", a, mem):
            kinds.add(x.kind)
            if x.tile >= 0:
                tiles.add(TILES[x.tile])
    assert kinds == {QUANTIZE, PACK, PARTIAL, PRODUCT, RESIDENT, JOIN}
    assert tiles >= {"256", "128", "64", "64x4", "loose64x4", "skinny64", "skinny16"}, tiles


def test_orthogonalize(lib):
    rng = random.Random(3)
    c = (ctypes.c_float * 18)(*([3.4445, -4.7750, 2.0315] * 6))
    tiles = set()
    for _ in range(300):
        it, ib = TYPES[rng.choice(list(TYPES))]
        ot, ob = TYPES[rng.choice(list(TYPES))]
        batch = rng.choice([1, 1, 2, 7])
        m, n = (rng.choice([1, 63, 64, 130, 515, 1500, 4096]) for _ in range(2))
        mem = Memory()
        a = _ffi.OrthogonalizeArgs(batch=batch, rows=m, cols=n, in_dtype=it, out_dtype=ot,
                                   steps=rng.choice([1, 2, 5, 6]), eps=1e-7, scale=1.0, keep=1.0,
                                   coefficients=ctypes.cast(c, c_void_p))

        def stack(eb, write=False):
            at, ld = mem.matrix(m, n, eb, rng, write)
            step = (m - 1) * ld + n + rng.choice([0, 5])
            mem.parts[-1] = (at, ((batch - 1) * step + (m - 1) * ld + n) * eb, write)
            return at, ld, step
        a.x, a.x_stride, a.x_batch_stride = stack(ib)
        a.out, a.out_stride, a.out_batch_stride = stack(ob, True)
        if rng.random() < 0.5:
            a.base, a.base_stride, a.base_batch_stride = stack(ob)
        got = run(lib, "lsamp_orthogonalize", a, mem)
        tiles |= {TILES[x.tile] for x in got if x.tile >= 0}
        assert [k for i, k in sorted({(x.launch, x.kind) for x in got})] == [START] + [
            GRAM, POLY, UPDATE] * a.steps
    assert tiles >= {"256", "192", "128", "64", "64x4", "32x8"}, tiles
