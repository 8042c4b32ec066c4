"""The launches that the hidden-state operators' C entry points make, without a
device: lsamp_head_api.cpp compiled over launches that are only written down
(head_launches.cpp)."""
from __future__ import annotations

import ctypes
import os
import subprocess
import tempfile
from ctypes import POINTER, byref, c_int32, c_int64, c_void_p

from lsamp import _ffi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "mlx-swift-lm_amd", "csrc")

(LINEAR, STATS, GRAD, STORE, PARTIAL, JOIN_LINEAR, JOIN_STORE, COL_SUM, COL_SUM_JOIN, PACK,
 JOIN_STATS, GRAD_SCALE, DROPOUT) = range(13)
TILES = ("256", "128", "64", "128x2", "64x4", "loose128", "loose64", "loose64x4", "skinny64",
         "skinny16")
ROLES = ("NT", "NN", "TN")
DTYPES = {"f32": (_ffi.DTYPE_F32, 4), "bf16": (_ffi.DTYPE_BF16, 2), "f16": (_ffi.DTYPE_F16, 2)}

_ints = ("kind tile roles parts m n slabs slabs_per_part accumulate first_col chunks stream element unused", c_int32)
_fields = [(f, c_int32) for f in _ints[0].split()]
_fields += [(f, c_int64) for f in "a a_ld b b_ld".split()]
_fields += [(f, c_int32) for f in "a_rows a_cols b_rows b_cols".split()]
_fields += [(f, c_int64) for f in "out ld_out out_bytes part_stride out2 out2_bytes".split()]


class Launch(ctypes.Structure):
    _fields_ = _fields


_lib = None


def lib():
    """The entry points over written-down launches, compiled once a process."""
    global _lib
    if _lib is None:
        with tempfile.TemporaryDirectory() as d:
            so = os.path.join(d, "head_launches.so")
            subprocess.run(
                ["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-w",
                 "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + CSRC,
                 os.path.join(CSRC, "lsamp_head_api.cpp"),
                 os.path.join(REPO, "tests", "head_launches.cpp"), "-o", so], check=True)
            _lib = ctypes.CDLL(so)
        assert _lib.head_launch_size() == ctypes.sizeof(Launch)
        _lib.head_launches.restype = c_int64
        for name, args in (("lsamp_linear", _ffi.LinearArgs),
                           ("lsamp_linear_backward", _ffi.LinearBackwardArgs),
                           ("lsamp_head_loss", _ffi.HeadLossArgs),
                           ("lsamp_head_loss_backward", _ffi.HeadLossBackwardArgs)):
            getattr(_lib, name).argtypes = [c_void_p, POINTER(args), c_void_p]
            getattr(_lib, name).restype = c_int32
            getattr(_lib, name + "_workspace").argtypes = [POINTER(args)]
            getattr(_lib, name + "_workspace").restype = c_int64
    return _lib


WORKSPACE = 1 << 44
AT = {n: (i + 1) << 50 for i, n in enumerate(
    "x weight bias residual out pre d_out d_x d_weight d_bias targets lse loss d_loss".split())}


def call(name, args):
    """(workspace bytes, launches) of the call; its workspace is at WORKSPACE."""
    L = lib()
    need = getattr(L, name + "_workspace")(byref(args))
    assert need >= 0, need
    args.workspace, args.workspace_bytes = WORKSPACE, need
    L.head_launches(None, 0)
    st = getattr(L, name)(1, byref(args), None)
    assert st == 0, st
    most = 4096
    out = (Launch * most)()
    n = L.head_launches(out, most)
    assert n <= most
    return need, out[:n]


def _bind(args, dtype, **matrices):
    """Pointers and strides: name -> columns, or (columns, stride, element offset)."""
    eb = DTYPES[dtype][1]
    for k, v in matrices.items():
        cols, stride, shift = v if isinstance(v, tuple) else (v, v, 0)
        setattr(args, k, AT[k] + shift * eb)
        setattr(args, k + "_stride", stride)
    return args


def _layout(cols, layout):
    """Row layouts of tests/head_common.py's matrix()."""
    return {"dense": (cols, cols, 0), "pad": (cols, cols + 8, 0), "odd": (cols, cols + 3, 1)}[layout]


def linear(dtype, m, k, n, layout="dense", *, pre=False, residual=False, out_f32=False):
    a = _ffi.LinearArgs(rows=m, in_features=k, out_features=n, dtype=DTYPES[dtype][0],
                        out_dtype=_ffi.DTYPE_F32 if out_f32 else DTYPES[dtype][0])
    _bind(a, dtype, x=_layout(k, layout), weight=_layout(k, layout), out=n)
    if residual:
        _bind(a, dtype, residual=n)
    if pre:
        a.pre, a.pre_stride = AT["pre"], n
    return call("lsamp_linear", a)


def linear_backward(dtype, m, k, n, layout="dense", *, activation=_ffi.ACT_NONE, bias=False,
                    want_x=True, want_weight=True):
    a = _ffi.LinearBackwardArgs(rows=m, in_features=k, out_features=n, dtype=DTYPES[dtype][0],
                                activation=activation, softcap=5.0)
    _bind(a, dtype, x=_layout(k, layout), weight=_layout(k, layout), d_out=_layout(n, layout))
    a.pre, a.pre_stride = AT["pre"], n
    if want_x:
        _bind(a, dtype, d_x=k)
    if want_weight:
        _bind(a, dtype, d_weight=k)
    if bias:
        a.d_bias = AT["d_bias"]
    return call("lsamp_linear_backward", a)


def head_loss(dtype, m, k, v, layout="dense"):
    a = _ffi.HeadLossArgs(rows=m, hidden=k, vocab=v, dtype=DTYPES[dtype][0])
    _bind(a, dtype, x=_layout(k, layout), weight=_layout(k, layout))
    a.targets, a.lse, a.loss = AT["targets"], AT["lse"], AT["loss"]
    return call("lsamp_head_loss", a)


def head_loss_backward(dtype, m, k, v, layout="dense", *, bias=False, want_x=True,
                       want_weight=True):
    a = _ffi.HeadLossBackwardArgs(rows=m, hidden=k, vocab=v, dtype=DTYPES[dtype][0])
    _bind(a, dtype, x=_layout(k, layout), weight=_layout(k, layout))
    a.targets, a.lse, a.d_loss = AT["targets"], AT["lse"], AT["d_loss"]
    if want_x:
        _bind(a, dtype, d_x=k)
    if want_weight:
        _bind(a, dtype, d_weight=k)
    if bias:
        a.d_bias = AT["d_bias"]
    return call("lsamp_head_loss_backward", a)


def check_workspace(need, launches):
    """Every write to the workspace ends inside it, buffers there do not overlap,
    and none is read before, or past what, it was written.  Sums of parts: what is added to was
    written before, every part written is joined, and the parts cover the
    reduction."""
    extent, written, chunks = {}, {}, {}
    for l in launches:
        for p, rows, ld, cols in ((l.a, l.a_rows, l.a_ld, l.a_cols), (l.b, l.b_rows, l.b_ld, l.b_cols)):
            if WORKSPACE <= p < min(AT.values()):
                assert p in extent, f"launch of kind {l.kind} reads what nothing has written"
                if l.element:
                    assert ((rows - 1) * ld + cols) * l.element <= extent[p], f"kind {l.kind} reads past {p}"
        for p, size in ((l.out, l.out_bytes), (l.out2, l.out2_bytes)):
            if size and WORKSPACE <= p < min(AT.values()):
                assert p + size <= WORKSPACE + need, (l.kind, p + size - WORKSPACE, need)
                extent[p] = max(extent.get(p, 0), size)
        if l.kind in (COL_SUM, GRAD) and l.out2:
            chunks[l.out2] = l.chunks
        if l.kind == COL_SUM_JOIN:
            assert l.chunks == chunks[l.a], "column sums left out"
        if l.kind == PARTIAL:
            assert l.parts * l.slabs_per_part >= l.slabs > (l.parts - 1) * l.slabs_per_part
            if l.accumulate:
                assert l.parts <= written[l.out], "added to parts that were never written"
            else:
                written[l.out] = l.parts
        if l.kind in (JOIN_LINEAR, JOIN_STORE):
            assert l.parts == written[l.a], "parts left out of the sum"
    end = 0
    for p in sorted(extent):
        assert p >= end, "buffers of the workspace overlap"
        end = p + extent[p]
