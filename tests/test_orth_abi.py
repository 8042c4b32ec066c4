"""CPU tests of lsamp_orthogonalize's arguments."""
from __future__ import annotations

import ctypes

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
