"""CPU tests of lsamp_orthogonalize's arguments."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from lsamp import _ffi

P = 0x10000  # (a device address that is never read here)


def workspace(coefficients=(3.4445, -4.7750, 2.0315), **kw):
    lib = _ffi.load_library()
    steps = kw.get("steps", 5)
    c = (ctypes.c_float * (3 * steps))(*(list(coefficients) * steps))
    a = _ffi.OrthogonalizeArgs(batch=1, rows=64, cols=64, in_dtype=_ffi.DTYPE_BF16,
                               out_dtype=_ffi.DTYPE_BF16, steps=steps,
                               coefficients=ctypes.cast(c, ctypes.c_void_p), eps=1e-7, scale=1.0,
                               keep=1.0, x=P, x_stride=64, out=P, out_stride=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.lsamp_orthogonalize_workspace(ctypes.byref(a))


@pytest.mark.parametrize("dtype", [_ffi.DTYPE_F32, _ffi.DTYPE_F16])
def test_fast_products_are_a_bfloat16_result_s(dtype):
    assert workspace(fast=1) > 0
    assert workspace(out_dtype=dtype) > 0
    assert workspace(out_dtype=dtype, fast=1) == _ffi.LSAMP_ERR_DTYPE
    assert workspace(fast=2) == _ffi.LSAMP_ERR_INVALID_ARGUMENT
    assert workspace(fast=-1) == _ffi.LSAMP_ERR_INVALID_ARGUMENT


def test_a_bfloat16_result_has_operands_of_two_parts():
    assert workspace() == workspace(out_dtype=_ffi.DTYPE_F32) > workspace(fast=1)


@pytest.mark.parametrize("c", [0.0, 1e-30, 1e-20, -1e-20, 1e-12, -1e-8, 1e-4])
def test_values_between_the_ends_are_bounded_for_any_last_coefficient(c):
    """100 s - 100 s^3 passes 38 at s = 0.58, also with a fifth power that is next to none."""
    assert workspace((100.0, -100.0, c), steps=1) == _ffi.LSAMP_ERR_INVALID_ARGUMENT
    assert workspace((20.0, -20.0, c), steps=1) > 0  # (7.7)
    assert workspace((20.0, -20.0, c), steps=2) == _ffi.LSAMP_ERR_INVALID_ARGUMENT


def test_bounds_are_those_of_a_fine_grid():
    """The largest |p| and |b t + c t^2| of a step, from their values at 200,001 places."""
    rng = np.random.default_rng(1)
    s = np.linspace(0, 1, 200001)
    for _ in range(300):
        a, b, c = (float(np.float32(v * 10.0 ** rng.uniform(-3, 1.2))) for v in rng.standard_normal(3))
        most = np.abs(a * s + b * s ** 3 + c * s ** 5).max()
        poly = np.abs(b * s ** 2 + c * s ** 4).max()
        # (a grid misses a maximum by half a step's square times the curvature, below 1e-8 here)
        if abs(most - 8) > 1e-6 and abs(poly - 128) > 1e-6:
            assert (workspace((a, b, c), steps=1) > 0) == (most < 8 and poly < 128), (a, b, c)
