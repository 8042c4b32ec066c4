"""Orthogonalised updates of matrices of any size against 64 bits, computed where the matrices
are, with check_orth's bound of blocks_common.py."""
from __future__ import annotations

import numpy as np
import torch

from blocks_common import orth_strict
from head_common import E, TINY, U

MUON = (3.4445, -4.7750, 2.0315)


def momenta(batch, rows, cols, dtype, seed, size=1e-3):
    """A falling spectrum above noise; many singular values are small."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")
    r = max(1, min(rows, cols) // 2)
    fall = 1 / (torch.arange(r, device="cuda") + 3.0)
    x = torch.stack([(randn(rows, r) * fall) @ randn(r, cols) + 0.02 * randn(rows, cols)
                     for _ in range(batch)])
    return (x * size).to(dtype)


def _halves(t, scale):
    h = (t * scale).half().double() / scale
    return h, ((t - h) * scale).half().double() / scale


def steps64(x, steps, coefficients=MUON, eps=1e-7, arithmetic="exact"):
    """A matrix's steps.  "exact": in 64 bits; "fast" and "full": with the roundings of
    products of one part and of two, sums in 64 bits (orth64's "f16" and "two")."""
    X = x.double()
    tall = X.shape[0] > X.shape[1]
    if tall:
        X = X.t().contiguous()
    norm = float(X.norm()) + float(np.float32(eps))
    a, b, c = (float(np.float32(v)) for v in coefficients)

    def times(l, r):  # of two parts each
        return l[0] @ (r[0] + r[1]) + l[1] @ r[0]

    if arithmetic != "fast":
        X = X / norm
    s = 1.0
    for i in range(steps):
        if arithmetic == "exact":
            A = X @ X.t().contiguous()
            X = a * X + (b * A + c * (A @ A)) @ X
        elif arithmetic == "full":
            x2 = _halves(X, 1024)
            A = _halves(times(x2, [v.t().contiguous() for v in x2]), 256)
            B = b * sum(A) + c * times(A, A)
            d = B.diagonal().clone()
            B.diagonal().zero_()
            X = (a + d)[:, None] * sum(x2) + times(_halves(B, 256), x2)
        else:
            if i == 0:
                e = 2.0 ** np.floor(np.log2(norm))
                X, s = X / e, e / norm
            h, lo = _halves(X, 1024)
            A = ((h @ h.t().contiguous()) * (s * s * 256)).half().double() / 256
            B = b * A + c * (A @ A)
            d = B.diagonal().clone()
            B.diagonal().zero_()
            X = s * ((a + d)[:, None] * (h + lo) + ((B * 256).half().double() / 256) @ h)
            s = 1.0
    return X.t() if tall else X


def check(got, x, steps, fast, coefficients=MUON, base=None, scale=1.0, keep=1.0, label=""):
    """Each matrix in the norm, as check_orth does from 32 x 32 on: at most twice what the
    emulated roundings are off by (two parts: and the float32 sums' share, sqrt(K) / 4 of
    them), the result's own rounding and those of scale and keep on top.  Smaller ones have
    few roundings, whose norm is not near its mean: orth_strict's bound.  Returns the largest
    error relative to the result's norm."""
    dt = got.dtype
    worst = 0.0
    for i in range(x.shape[0]):
        want = steps64(x[i], steps, coefficients)
        if min(want.shape) < 32:
            bound = orth_strict(x[i], steps, coefficients, 1e-7, fast)
        else:
            model = steps64(x[i], steps, coefficients, arithmetic="fast" if fast else "full")
            sums = 0.0 if fast else np.sqrt(max(want.shape)) / 4
            bound = float((model - want).norm()) * (2.0 + sums)
        kept = keep * base[i].double() if base is not None else torch.zeros_like(want)
        y = scale * want + kept
        bound = (abs(scale) * bound + U[dt] * (float(y.norm()) + abs(scale) * bound)
                 + 3 * E * (abs(scale) * float(want.norm()) + float(kept.norm()))
                 + TINY[dt] * U[dt] * y.numel() ** 0.5)
        far = float((got[i].double() - y).norm())
        assert far <= bound, f"{label} matrix {i}: {far:.3g} off, {bound:.3g} allowed"
        worst = max(worst, far / float(y.norm()))
    return worst
