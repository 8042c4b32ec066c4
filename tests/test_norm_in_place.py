"""CPU test of a norm's gradients that are written over what they are taken from: the columns'
sums are then not taken in the same launch, by work-groups that read what others overwrite, but
as shares in the workspace."""
from __future__ import annotations

import ctypes

import pytest

from lsamp import _ffi

X, D, R, OUT, V = (0x100000 * (i + 1) for i in range(5))  # (addresses that are never read here)


@pytest.mark.parametrize("rows", [4, 768])
@pytest.mark.parametrize("dtype", [_ffi.DTYPE_F32, _ffi.DTYPE_BF16, _ffi.DTYPE_F16])
def test_sums_of_few_rows(rows, dtype):
    def workspace(d_x, d_weight=V):
        a = _ffi.LayerNormBackwardArgs(rows=rows, cols=64, dtype=dtype, x=X, x_stride=64, mean=V,
                                       rstd=V, d_out=D, d_out_stride=64, residual=R if d_x else None,
                                       residual_stride=64, d_x=d_x, d_x_stride=64, d_weight=d_weight)
        return _ffi.load_library().lsamp_layer_norm_backward_workspace(ctypes.byref(a))
    assert workspace(OUT) == workspace(R) == workspace(None) == 0
    assert workspace(D) > 0 and workspace(X) == workspace(D)
    assert workspace(X, d_weight=None) == 0
