"""Prepared calls of the hidden-state operators (include/lsamp.h): linear
blocks, the vocabulary head's cross entropy, their gradients, and dropout.

Made by the Context methods of the same names (`Context.prepare_linear`, ...).
A prepared call holds its inputs, outputs and workspace; `launch()` is one C
call on the current torch stream (or the one given) and can be captured in a
HIP graph.  Inputs are read at each launch, so a training loop writes the next
batch into the same tensors.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _ffi

ACTIVATIONS = {"none": _ffi.ACT_NONE, "relu": _ffi.ACT_RELU, "silu": _ffi.ACT_SILU,
               "gelu": _ffi.ACT_GELU, "gelu_tanh": _ffi.ACT_GELU_TANH,
               "softcap": _ffi.ACT_SOFTCAP}
DTYPES = {torch.float32: _ffi.DTYPE_F32, torch.bfloat16: _ffi.DTYPE_BF16,
          torch.float16: _ffi.DTYPE_F16}


def _activation(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    return ACTIVATIONS[name]


def _stream_of(device: torch.device) -> int:
    """The current torch stream's handle (without the 2 us of building a
    torch.cuda.Stream, as long as a small launch itself)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device.index) if raw else torch.cuda.current_stream(device).cuda_stream


class PreparedCall:
    """One bound C call; `keep_alive` holds every tensor whose pointer it has."""

    entry = ""

    def __init__(self, ctx, device):
        self.ctx = ctx
        self.device = device
        if device != torch.device("cuda", ctx.device):
            raise ValueError(f"tensors are on {device}, the context on cuda:{ctx.device}")
        self.keep_alive = []
        self.args = None
        self.stream = _stream_of(device)

    # ------------------------------------------------------------- arguments
    def _matrix(self, name: str, t: torch.Tensor, rows: Optional[int] = None,
                cols: Optional[int] = None, dtype: Optional[torch.dtype] = None):
        """(pointer, row stride) of a [rows, cols] view with dense rows."""
        if t.dim() != 2 or (rows is not None and t.shape[0] != rows) or (
                cols is not None and t.shape[1] != cols):
            raise ValueError(f"{name} must be [{rows or 'rows'}, {cols or 'columns'}], "
                             f"got {tuple(t.shape)}")
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"{name} rows must be contiguous")
        if dtype is not None and t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
        if t.dtype not in DTYPES:
            raise ValueError(f"{name}: {t.dtype} is not float32, bfloat16 or float16")
        if t.device != self.device:
            raise ValueError(f"{name} must be on {self.device}")
        self.keep_alive.append(t)
        return t.data_ptr(), t.stride(0)

    def _vector(self, name: str, t: torch.Tensor, n: int, dtype: torch.dtype):
        if t.dim() != 1 or t.shape[0] != n or t.dtype != dtype or (n > 1 and t.stride(0) != 1):
            raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n}")
        if t.device != self.device:
            raise ValueError(f"{name} must be on {self.device}")
        self.keep_alive.append(t)
        return t.data_ptr()

    def _empty(self, shape, dtype):
        t = torch.empty(shape, dtype=dtype, device=self.device)
        self.keep_alive.append(t)
        return t

    def _bind(self, args):
        """Sizes and allocates the workspace of the finished arguments."""
        self.args = args
        self._byref = ctypes.byref(args)
        self._entry = getattr(self.ctx.lib, self.entry)
        if hasattr(args, "workspace_bytes"):
            need = getattr(self.ctx.lib, self.entry + "_workspace")(self._byref)
            if need < 0:
                raise _ffi.LsampError(int(need), self.entry)
            if need:
                self.workspace = self._empty(need, torch.uint8)
                args.workspace = self.workspace.data_ptr()
                args.workspace_bytes = need

    def launch(self, stream: Optional[int] = None) -> None:
        s = stream if stream is not None else _stream_of(self.device)
        if s != self.stream:
            # the allocator must not hand these out while this stream reads them
            ext = torch.cuda.ExternalStream(s, device=self.device)
            for t in self.keep_alive:
                t.record_stream(ext)
        st = self._entry(self.ctx.handle, self._byref, s)
        if st != 0:
            raise _ffi.LsampError(st, self.entry)

    def outputs(self) -> dict:
        raise NotImplementedError


class PreparedLinear(PreparedCall):
    """out = act(x weight^T + bias) + residual (lsamp_linear); `pre` holds
    x weight^T + bias in float32 where asked for."""

    entry = "lsamp_linear"

    def __init__(self, ctx, x, weight, *, bias=None, residual=None, activation="none",
                 softcap=0.0, out_dtype=None, want_pre=False, out=None):
        super().__init__(ctx, x.device)
        a = _ffi.LinearArgs()
        a.x, a.x_stride = self._matrix("x", x)
        rows, k = x.shape
        a.weight, a.weight_stride = self._matrix("weight", weight, cols=k, dtype=x.dtype)
        n = weight.shape[0]
        a.rows, a.in_features, a.out_features = rows, k, n
        a.dtype = DTYPES[x.dtype]
        a.activation, a.softcap = _activation(activation), softcap
        out_dtype = (out.dtype if out is not None else x.dtype) if out_dtype is None else out_dtype
        if out_dtype not in (x.dtype, torch.float32):
            raise ValueError(f"out_dtype must be {x.dtype} or float32")
        a.out_dtype = DTYPES[out_dtype]
        if bias is not None:
            a.bias = self._vector("bias", bias, n, x.dtype)
        if residual is not None:
            a.residual, a.residual_stride = self._matrix("residual", residual, rows, n, x.dtype)
        self.out = self._empty((rows, n), out_dtype) if out is None else out
        a.out, a.out_stride = self._matrix("out", self.out, rows, n, out_dtype)
        self.pre = self._empty((rows, n), torch.float32) if want_pre else None
        if want_pre:
            a.pre, a.pre_stride = self.pre.data_ptr(), n
        self._bind(a)

    def outputs(self) -> dict:
        return {"out": self.out} if self.pre is None else {"out": self.out, "pre": self.pre}


class PreparedLinearBackward(PreparedCall):
    """The gradients of a linear call at d_out (lsamp_linear_backward)."""

    entry = "lsamp_linear_backward"

    def __init__(self, ctx, d_out, x, weight, *, pre=None, activation="none", softcap=0.0,
                 want_x=True, want_weight=True, want_bias=False):
        super().__init__(ctx, d_out.device)
        a = _ffi.LinearBackwardArgs()
        rows, k = x.shape
        n = weight.shape[0]
        a.d_out, a.d_out_stride = self._matrix("d_out", d_out, rows, n)
        dt = d_out.dtype
        a.x, a.x_stride = self._matrix("x", x, dtype=dt)
        a.weight, a.weight_stride = self._matrix("weight", weight, n, k, dt)
        a.rows, a.in_features, a.out_features = rows, k, n
        a.dtype = DTYPES[dt]
        a.activation, a.softcap = _activation(activation), softcap
        if pre is not None:
            a.pre, a.pre_stride = self._matrix("pre", pre, rows, n, torch.float32)
        self.d_x = self._empty((rows, k), dt) if want_x else None
        self.d_weight = self._empty((n, k), dt) if want_weight else None
        self.d_bias = self._empty(n, dt) if want_bias else None
        if want_x:
            a.d_x, a.d_x_stride = self.d_x.data_ptr(), k
        if want_weight:
            a.d_weight, a.d_weight_stride = self.d_weight.data_ptr(), k
        if want_bias:
            a.d_bias = self.d_bias.data_ptr()
        self._bind(a)

    def outputs(self) -> dict:
        o = {"d_x": self.d_x, "d_weight": self.d_weight, "d_bias": self.d_bias}
        return {k: v for k, v in o.items() if v is not None}


class PreparedHeadLoss(PreparedCall):
    """Cross entropy of the vocabulary head over hidden states x
    (lsamp_head_loss): loss and log-sum-exp of every row, row flags."""

    entry = "lsamp_head_loss"

    def __init__(self, ctx, x, weight, targets, *, bias=None, softcap=0.0):
        super().__init__(ctx, x.device)
        a = _ffi.HeadLossArgs()
        a.x, a.x_stride = self._matrix("x", x)
        rows, k = x.shape
        a.weight, a.weight_stride = self._matrix("weight", weight, cols=k, dtype=x.dtype)
        a.rows, a.hidden, a.vocab = rows, k, weight.shape[0]
        a.dtype, a.softcap = DTYPES[x.dtype], softcap
        if bias is not None:
            a.bias = self._vector("bias", bias, a.vocab, x.dtype)
        a.targets = self._vector("targets", targets, rows, torch.int32)
        self.loss = self._empty(rows, torch.float32)
        self.lse = self._empty(rows, torch.float32)
        self.row_flags = self._empty(rows, torch.int32)
        a.loss, a.lse = self.loss.data_ptr(), self.lse.data_ptr()
        a.row_flags = self.row_flags.data_ptr()
        self._bind(a)

    def outputs(self) -> dict:
        return {"loss": self.loss, "lse": self.lse, "row_flags": self.row_flags}


class PreparedHeadLossBackward(PreparedCall):
    """The gradients of sum_r d_loss[r] loss[r] (lsamp_head_loss_backward);
    `lse` is the forward call's."""

    entry = "lsamp_head_loss_backward"

    def __init__(self, ctx, d_loss, x, weight, targets, *, lse, bias=None, softcap=0.0,
                 want_x=True, want_weight=True, want_bias=False):
        super().__init__(ctx, x.device)
        a = _ffi.HeadLossBackwardArgs()
        a.x, a.x_stride = self._matrix("x", x)
        rows, k = x.shape
        a.weight, a.weight_stride = self._matrix("weight", weight, cols=k, dtype=x.dtype)
        v = weight.shape[0]
        a.rows, a.hidden, a.vocab = rows, k, v
        a.dtype, a.softcap = DTYPES[x.dtype], softcap
        if bias is not None:
            a.bias = self._vector("bias", bias, v, x.dtype)
        a.targets = self._vector("targets", targets, rows, torch.int32)
        a.lse = self._vector("lse", lse, rows, torch.float32)
        a.d_loss = self._vector("d_loss", d_loss, rows, torch.float32)
        self.d_x = self._empty((rows, k), x.dtype) if want_x else None
        self.d_weight = self._empty((v, k), x.dtype) if want_weight else None
        self.d_bias = self._empty(v, x.dtype) if want_bias else None
        if want_x:
            a.d_x, a.d_x_stride = self.d_x.data_ptr(), k
        if want_weight:
            a.d_weight, a.d_weight_stride = self.d_weight.data_ptr(), k
        if want_bias:
            a.d_bias = self.d_bias.data_ptr()
        self._bind(a)

    def outputs(self) -> dict:
        o = {"d_x": self.d_x, "d_weight": self.d_weight, "d_bias": self.d_bias}
        return {k: v for k, v in o.items() if v is not None}


class PreparedDropout(PreparedCall):
    """out = residual + dropout(x) (lsamp_dropout).  The same key, offset and
    p drop the same elements: the backward pass is this call on the gradient.
    `step` (an int64 device tensor of one element) is added to the offset, so the
    offsets of layers lie further apart than any step (layer << 48)."""

    entry = "lsamp_dropout"

    def __init__(self, ctx, x, *, p, key, offset=0, residual=None, step=None, out=None):
        super().__init__(ctx, x.device)
        a = _ffi.DropoutArgs()
        a.x, a.x_stride = self._matrix("x", x)
        a.rows, a.cols = x.shape
        a.dtype, a.p = DTYPES[x.dtype], p
        a.key, a.offset = key % (1 << 64), offset % (1 << 64)
        if step is not None:
            a.step = self._vector("step", step, 1, torch.int64)
        if residual is not None:
            a.residual, a.residual_stride = self._matrix("residual", residual, *x.shape, x.dtype)
        self.out = self._empty(tuple(x.shape), x.dtype) if out is None else out
        a.out, a.out_stride = self._matrix("out", self.out, *x.shape, x.dtype)
        self._bind(a)

    def outputs(self) -> dict:
        return {"out": self.out}
