"""CPU tests of the C ABI of a block's other operators: struct layouts,
workspace sizes (host arithmetic, no device needed) and refusals."""
from __future__ import annotations

import ctypes

import pytest

from lsamp import _ffi

P = 0x10000  # (a device address that is never read here)
I, S, D = _ffi.LSAMP_ERR_INVALID_ARGUMENT, _ffi.LSAMP_ERR_SHAPE, _ffi.LSAMP_ERR_DTYPE


@pytest.fixture(scope="module")
def lib():
    return _ffi.load_library()


@pytest.mark.parametrize("name,struct", [
    ("lsamp_layer_norm_args", _ffi.LayerNormArgs),
    ("lsamp_layer_norm_backward_args", _ffi.LayerNormBackwardArgs),
    ("lsamp_quantize_rows_args", _ffi.QuantizeRowsArgs),
    ("lsamp_linear_int8_args", _ffi.LinearInt8Args),
    ("lsamp_orthogonalize_args", _ffi.OrthogonalizeArgs)])
def test_struct_layouts_agree(lib, name, struct):
    assert lib.lsamp_abi_sizeof(name.encode()) == ctypes.sizeof(struct)


def _set(a, kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def norm_backward(lib, **kw):
    a = _ffi.LayerNormBackwardArgs(rows=4, cols=64, dtype=_ffi.DTYPE_BF16, x=P, x_stride=64, mean=P,
                                   rstd=P, d_out=P, d_out_stride=64, d_x=P, d_x_stride=64,
                                   d_weight=P, d_bias=P)
    return lib.lsamp_layer_norm_backward_workspace(_set(a, kw))


def int8(lib, **kw):
    a = _ffi.LinearInt8Args(rows=4, in_features=64, out_features=32, dtype=_ffi.DTYPE_BF16,
                            activation=_ffi.ACT_NONE, out_dtype=_ffi.DTYPE_BF16, x=P, x_stride=64,
                            weight=P, weight_stride=64, weight_scale=P, out=P, out_stride=32)
    return lib.lsamp_linear_int8_workspace(_set(a, kw))


def orth(lib, coefficients=(3.4445, -4.7750, 2.0315), **kw):
    steps = kw.get("steps", 5)
    c = (ctypes.c_float * (3 * max(1, steps)))(*(list(coefficients) * max(1, steps)))
    a = _ffi.OrthogonalizeArgs(batch=1, rows=64, cols=64, in_dtype=_ffi.DTYPE_BF16,
                               out_dtype=_ffi.DTYPE_BF16, steps=steps,
                               coefficients=ctypes.cast(c, ctypes.c_void_p), eps=1e-7, scale=1.0,
                               keep=1.0, x=P, x_stride=64, out=P, out_stride=64)
    return lib.lsamp_orthogonalize_workspace(_set(a, kw))


def test_norm_backward_refusals(lib):
    assert lib.lsamp_layer_norm_backward_workspace(None) == I
    assert norm_backward(lib) >= 0
    assert norm_backward(lib, d_weight=None, d_bias=None) == 0
    for kw, want in [(dict(rows=0), S), (dict(cols=0), S), (dict(cols=(1 << 22) + 1), S),
                     (dict(dtype=3), D), (dict(x=None), I), (dict(x=P + 1), I),
                     (dict(d_out=None), I), (dict(mean=None), I), (dict(rstd=P + 2), I),
                     (dict(x_stride=63), S), (dict(d_x_stride=63), S), (dict(weight=P + 1), I),
                     (dict(residual=P, residual_stride=63), S),
                     (dict(residual=P, residual_stride=64, d_x=None), I),
                     (dict(d_x=None, d_weight=None, d_bias=None), I)]:
        assert norm_backward(lib, **kw) == want, kw
        assert lib.lsamp_last_error()


def test_norm_backward_workspace(lib):
    """Two float32 sums of every column for each work-group: at most 512 of them."""
    assert norm_backward(lib, rows=1 << 20, cols=4096, x_stride=4096, d_out_stride=4096,
                         d_x_stride=4096) <= 512 * 2 * 4096 * 4
    assert norm_backward(lib, rows=2000) >= 2 * 64 * 4


def test_linear_int8_refusals(lib):
    assert lib.lsamp_linear_int8_workspace(None) == I
    assert int8(lib, rows=1) == 0 and int8(lib, rows=8) >= 8 * 64 + 8 * 4
    # (few rows are kept on the chip in rows of multiples of 256 bytes)
    assert int8(lib, x_scale=P, in_features=256, x_stride=256, weight_stride=256) == 0
    assert int8(lib, x_scale=P) >= 4 * 256
    for kw, want in [(dict(rows=0), S), (dict(in_features=0), S), (dict(out_features=0), S),
                     (dict(in_features=131072, x_stride=131072, weight_stride=131072), S),
                     (dict(dtype=3), D), (dict(out_dtype=_ffi.DTYPE_F16), D),
                     (dict(activation=6), I), (dict(activation=_ffi.ACT_SOFTCAP), I),
                     (dict(x=None), I), (dict(weight=None), I), (dict(weight_scale=None), I),
                     (dict(weight_scale=P + 2), I), (dict(x_scale=P + 2), I), (dict(out=None), I),
                     (dict(x=P + 1), I), (dict(x_stride=63), S), (dict(weight_stride=63), S),
                     (dict(out_stride=31), S), (dict(bias=P + 1), I),
                     (dict(residual=P, residual_stride=31), S)]:
        assert int8(lib, **kw) == want, kw
        assert lib.lsamp_last_error()
    assert int8(lib, x=P + 1, x_scale=P) >= 0  # (bytes lie anywhere)


def test_orthogonalize_refusals(lib):
    assert lib.lsamp_orthogonalize_workspace(None) == I
    assert orth(lib) > 0
    inf = float("inf")
    for kw, want in [(dict(batch=0), S), (dict(batch=65536), S), (dict(rows=0), S), (dict(cols=-1), S),
                     (dict(in_dtype=3), D), (dict(out_dtype=-1), D), (dict(steps=0), I),
                     (dict(steps=65), I), (dict(eps=0.0), I), (dict(eps=inf), I),
                     (dict(scale=inf), I), (dict(keep=inf), I), (dict(x=None), I),
                     (dict(out=None), I), (dict(x=P + 1), I), (dict(x_stride=63), S),
                     (dict(out_stride=63), S), (dict(base=P, base_stride=63), S),
                     (dict(batch=2, out_batch_stride=64 * 64 - 1), S),
                     (dict(batch=2, out_batch_stride=64 * 64, x_batch_stride=-1), S),
                     (dict(rows=1 << 22, cols=1 << 22, x_stride=1 << 22, out_stride=1 << 22), S),
                     (dict(coefficients=(3.5, 4.8, 2.0)), I),
                     (dict(coefficients=(9.0, -9.0, 8.0)), I),
                     (dict(coefficients=(float("nan"), 0.0, 0.0)), I)]:
        assert orth(lib, **kw) == want, kw
        assert lib.lsamp_last_error()
    assert orth(lib, coefficients=(1.5, -0.5, 0.0), steps=20) > 0
    assert orth(lib, coefficients=(1.0, 0.0, 0.0)) > 0


def test_orthogonalize_bounds_the_values(lib):
    """A cubic that grows only between its ends is found: 8.2 s - 8 s^3 ends at 0.2 but
    passes 3.2 on the way, and the next steps leave (0, 8)."""
    assert orth(lib, coefficients=(8.2, -8.0, 0.0), steps=1) > 0
    assert orth(lib, coefficients=(8.2, -8.0, 0.0), steps=3) == I
