"""CPU tests of the hidden-state operators' C ABI: struct layouts, workspace
sizes (host arithmetic, no device needed) and refusals."""
from __future__ import annotations

import ctypes

import pytest

from lsamp import _ffi


@pytest.fixture(scope="module")
def lib():
    return _ffi.load_library()


@pytest.mark.parametrize("name,struct", [
    ("lsamp_linear_args", _ffi.LinearArgs),
    ("lsamp_linear_backward_args", _ffi.LinearBackwardArgs),
    ("lsamp_head_loss_args", _ffi.HeadLossArgs),
    ("lsamp_head_loss_backward_args", _ffi.HeadLossBackwardArgs),
    ("lsamp_dropout_args", _ffi.DropoutArgs)])
def test_struct_layouts_agree(lib, name, struct):
    assert lib.lsamp_abi_sizeof(name.encode()) == ctypes.sizeof(struct)


P = 0x10000  # (a device address that is never read here)


def linear(**kw):
    a = _ffi.LinearArgs(rows=4, in_features=64, out_features=32, dtype=_ffi.DTYPE_BF16,
                        activation=_ffi.ACT_NONE, out_dtype=_ffi.DTYPE_BF16, x=P, x_stride=64,
                        weight=P, weight_stride=64, out=P, out_stride=32)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def loss(cls=_ffi.HeadLossArgs, **kw):
    a = cls(rows=300, hidden=64, vocab=5000, dtype=_ffi.DTYPE_BF16, x=P, x_stride=64, weight=P,
            weight_stride=64, targets=P, lse=P)
    if cls is _ffi.HeadLossArgs:
        a.loss = P
    else:
        a.d_loss, a.d_x, a.d_x_stride, a.d_weight, a.d_weight_stride = P, P, 64, P, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_linear_refusals(lib):
    f = lambda **kw: lib.lsamp_linear_workspace(ctypes.byref(linear(**kw)))  # noqa: E731
    assert f() >= 0
    I, S, D = _ffi.LSAMP_ERR_INVALID_ARGUMENT, _ffi.LSAMP_ERR_SHAPE, _ffi.LSAMP_ERR_DTYPE
    assert lib.lsamp_linear_workspace(None) == I
    for kw, want in [(dict(rows=0), S), (dict(rows=-1), S), (dict(in_features=0), S),
                     (dict(out_features=0), S), (dict(rows=1 << 28), S), (dict(dtype=3), D),
                     (dict(out_dtype=_ffi.DTYPE_F16), D), (dict(activation=6), I),
                     (dict(activation=-1), I), (dict(activation=_ffi.ACT_SOFTCAP), I),
                     (dict(x=None), I), (dict(weight=None), I), (dict(out=None), I),
                     (dict(x_stride=63), S), (dict(weight_stride=63), S), (dict(out_stride=31), S),
                     (dict(x=P + 1), I), (dict(bias=P + 1), I), (dict(pre=P + 2, pre_stride=32), I),
                     (dict(residual=P, residual_stride=31), S), (dict(x_stride=-64), S),
                     (dict(x_stride=1 << 41), S)]:
        assert f(**kw) == want, kw
        assert lib.lsamp_last_error()


def test_linear_workspace_counts_alignment(lib):
    f = lambda **kw: lib.lsamp_linear_workspace(ctypes.byref(linear(**kw)))  # noqa: E731
    big = dict(rows=8192, in_features=4096, out_features=4096, weight_stride=4096,
               out_stride=4096, x_stride=4096)
    base, copy = f(**big), 8192 * 4096 * 2
    # rows that start between 16-byte chunks are copied; so are rows too far apart
    assert f(**dict(big, x=P + 2)) >= base + copy
    assert f(**dict(big, x_stride=4097)) >= base + copy
    assert f(**dict(big, x_stride=1 << 30)) >= base + copy
    assert f(**dict(big, x_stride=4104)) == base
    # small and few rows are read as they are
    assert f(rows=100, x=P + 2, x_stride=65) == f(rows=100)
    assert f(x=P + 2, x_stride=65) == 0
    assert f(rows=1, x_stride=1) == 0  # (a one-row matrix carries any stride)


@pytest.mark.parametrize("cls,entry", [
    (_ffi.HeadLossArgs, "lsamp_head_loss"),
    (_ffi.HeadLossBackwardArgs, "lsamp_head_loss_backward")])
def test_head_loss_refusals(lib, cls, entry):
    ws = getattr(lib, entry + "_workspace")
    f = lambda **kw: ws(ctypes.byref(loss(cls, **kw)))  # noqa: E731
    assert f() > 0
    I, S, D = _ffi.LSAMP_ERR_INVALID_ARGUMENT, _ffi.LSAMP_ERR_SHAPE, _ffi.LSAMP_ERR_DTYPE
    assert ws(None) == I
    for kw, want in [(dict(rows=0), S), (dict(hidden=0), S), (dict(vocab=0), S), (dict(dtype=7), D),
                     (dict(softcap=-1.0), I), (dict(softcap=float("inf")), I),
                     (dict(softcap=float("nan")), I), (dict(x=None), I), (dict(weight=None), I),
                     (dict(targets=None), I), (dict(targets=P + 2), I), (dict(lse=None), I),
                     (dict(x_stride=10), S), (dict(weight_stride=10), S)]:
        assert f(**kw) == want, kw
    if cls is _ffi.HeadLossBackwardArgs:
        assert f(d_loss=None) == I
        assert f(d_x=None, d_weight=None) == I
        assert f(d_x_stride=63) == S and f(d_weight_stride=63) == S
    else:
        assert f(loss=None) == I


def test_head_loss_workspace_stays_small(lib):
    """A long training batch over a large vocabulary: no logits of 4,096 x
    151,936 are held, only a piece of their gradient and d_x's float32 sums."""
    a = loss(_ffi.HeadLossBackwardArgs, rows=4096, hidden=4096, vocab=151936, x_stride=4096,
             weight_stride=4096, d_x_stride=4096, d_weight_stride=4096)
    need = lib.lsamp_head_loss_backward_workspace(ctypes.byref(a))
    assert 0 < need < 4096 * 151936 * 2 / 3
    a = loss(rows=4096, hidden=4096, vocab=151936, x_stride=4096, weight_stride=4096)
    need = lib.lsamp_head_loss_workspace(ctypes.byref(a))
    assert 0 < need < 4096 * 151936 * 2 / 16


def test_calls_without_a_context(lib):
    a = linear()
    assert lib.lsamp_linear(None, ctypes.byref(a), None) == _ffi.LSAMP_ERR_INVALID_ARGUMENT
    assert b"context" in lib.lsamp_last_error()
    for entry in ("lsamp_linear_backward", "lsamp_head_loss", "lsamp_head_loss_backward",
                  "lsamp_dropout"):
        assert getattr(lib, entry)(None, None, None) == _ffi.LSAMP_ERR_INVALID_ARGUMENT


def test_limits_of_sizes(lib):
    """A tile's rows lie within 32 bits of its first: features end at 2^22; a
    loss has a work-group a row: 2^23 rows."""
    wide = 1 << 22
    f = lambda **kw: lib.lsamp_linear_workspace(ctypes.byref(linear(**kw)))  # noqa: E731
    S = _ffi.LSAMP_ERR_SHAPE
    for dtype in (_ffi.DTYPE_F32, _ffi.DTYPE_BF16):
        kw = dict(rows=100, dtype=dtype, out_dtype=dtype)
        assert f(in_features=wide, x_stride=wide, weight_stride=wide, **kw) >= 0
        assert f(in_features=wide + 1, x_stride=wide + 1, weight_stride=wide + 1, **kw) == S
        assert f(out_features=wide, out_stride=wide, **kw) >= 0
        assert f(out_features=wide + 1, out_stride=wide + 1, **kw) == S
    for cls, entry in ((_ffi.HeadLossArgs, lib.lsamp_head_loss_workspace),
                       (_ffi.HeadLossBackwardArgs, lib.lsamp_head_loss_backward_workspace)):
        assert entry(ctypes.byref(loss(cls, rows=1 << 23))) > 0
        assert entry(ctypes.byref(loss(cls, rows=(1 << 23) + 1))) == S
        assert b"rows" in lib.lsamp_last_error()
        assert entry(ctypes.byref(loss(cls, vocab=wide + 1))) == S
