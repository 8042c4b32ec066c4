"""64-bit restatements of a block's other operators (lsamp_layer_norm,
lsamp_quantize_rows, lsamp_linear_int8, lsamp_orthogonalize and the norm's
gradients), each with a bound on what the kernels' arithmetic may be off by.

As in head_common, the bounds are worst cases of the promised arithmetic,
element by element, with U a type's unit roundoff and E float32's.  A row's sums
are added in a tree: a thread's 8 V values one after the other (V groups of
eight; of rows past 16,384 elements, cols / 1024 more), six exchanges within a
wave and at most 16 waves, so at most `depth` roundings meet a value, not cols.
"""
from __future__ import annotations

import numpy as np
import torch

from head_common import E, TINY, U, act64, d64


def depth(cols):
    return 64 + (cols // 1024 if cols > 16384 else 0)


def rounded(y, err, dt):
    return y, err + U[dt] * (y.abs() + err) + TINY[dt] * U[dt]


def norm64(x, weight, bias, eps):
    X = d64(x)
    n = X.shape[1]
    D = depth(n)
    eps = float(np.float32(eps))
    mean = X.mean(1, keepdim=True)
    c = X - mean
    var = (c * c).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    # the mean: D roundings of the sum, two of the product with 1 / cols
    dm = (D + 1) * E * X.abs().mean(1, keepdim=True) + 2 * E * mean.abs()
    # the variance around a mean that is dm off is larger by dm^2; each square is rounded
    # with its difference (three times E), then added up, divided, eps added
    rel = 0.5 * ((D + 8) * E + dm * dm / (var + eps)) + 4 * E
    xh = c * rstd
    err = rstd * (dm + E * c.abs()) + xh.abs() * (rel + 2 * E)
    y = xh
    if weight is not None:
        w = d64(weight)
        y, err = y * w, err * w.abs() + E * (y * w).abs()
    if bias is not None:
        y = y + d64(bias)
        err = err + E * (y.abs() + err)
    out = rounded(y, err, x.dtype)
    return {"out": out, "mean": (mean[:, 0], dm[:, 0]), "rstd": (rstd[:, 0], (rstd * rel)[:, 0])}


def norm_grads64(d_out, x, mean, rstd, weight, residual):
    """From the kernel's own mean and rstd (float32), as the operator is defined."""
    dt = x.dtype
    X, d = d64(x), d64(d_out)
    rows, n = X.shape
    D = depth(n)
    mu, r = d64(mean)[:, None], d64(rstd)[:, None]
    xh = (X - mu) * r
    dxh = 2 * E * xh.abs()
    w = torch.ones(n, dtype=torch.float64) if weight is None else d64(weight)
    g = d * w
    c1 = g.mean(1, keepdim=True)
    c2 = (g * xh).mean(1, keepdim=True)
    e1 = (D + 4) * E * g.abs().mean(1, keepdim=True)
    e2 = (D + 8) * E * (g * xh).abs().mean(1, keepdim=True)
    y = r * (g - c1 - xh * c2)
    err = r * (E * g.abs() + e1 + xh.abs() * e2 + dxh * c2.abs()
               + 4 * E * (g.abs() + c1.abs() + (xh * c2).abs()))
    if residual is not None:
        y = y + d64(residual)
        err = err + E * (y.abs() + err)
    # a column's sum: a work-group's rows one after the other (at most rows / 256, or 64 of
    # long rows), its waves, then at most 512 shares in sixteen waves
    R = 64 + rows // 256 + 64
    dw = (d * xh).sum(0)
    dw_err = (R + 4) * E * (d * xh).abs().sum(0)
    db = d.sum(0)
    db_err = R * E * d.abs().sum(0)
    return {"d_x": rounded(y, err, dt), "d_weight": rounded(dw, dw_err, dt),
            "d_bias": rounded(db, db_err, dt)}


def quantize64(x):
    """(q, scale), exactly."""
    a = d64(x).numpy()
    finite = np.isfinite(a).all(1)
    top = np.where(finite, np.abs(np.where(np.isfinite(a), a, 0)).max(1), 0).astype(np.float32)
    part = np.float32(1) / np.float32(127)
    scale = np.maximum(top * part, np.float32(2.0 ** -126))
    # (24-bit by 24-bit quotients below 128: no rounding to 53 bits reaches a tie)
    q = np.clip(np.rint(np.where(np.isfinite(a), a, 0) / scale.astype(np.float64)[:, None]), -127, 127)
    q[~finite] = 0
    scale = scale.copy()
    scale[~finite] = np.nan
    return torch.from_numpy(q).to(torch.int8), torch.from_numpy(scale)


def int8_64(q, scale, w, w_scale, bias=None, residual=None, act="none", cap=0.0, dtype=None,
            out_dtype=None):
    """Whole sums are exact; a sum becomes float32, its scales are multiplied, and the
    two with each other: three roundings."""
    out_dtype = out_dtype or dtype
    z = (q.cpu().double() @ w.cpu().double().t()) * d64(scale)[:, None] * d64(w_scale)
    err = 3 * E * z.abs()
    if bias is not None:
        z = z + d64(bias)
        err = err + E * (z.abs() + err)
    y, _ = act64(act, z, cap)
    if act != "none":  # (as in linear64)
        err = 1.2 * err + 16 * E * (z.abs() + 1)
    if residual is not None:
        y = y + d64(residual)
        err = err + E * (y.abs() + err)
    return rounded(y, err, out_dtype)


def _two_parts(t, scale):
    h = (t * scale).half().double() / scale
    return h, ((t - h) * scale).half().double() / scale


def orth64(x, steps, coefficients, eps, arithmetic="exact"):
    """One matrix.  "exact": in 64 bits.  "f16": with the roundings that a bfloat16 result's
    steps make (X in two float16 parts of which products take the first, A and B in
    float16, B's diagonal apart; sums in 64 bits).  "two": with those of float32 and float16
    results (X, A and B in two float16 parts, whose last products are left out)."""
    G = d64(x)
    tall = G.shape[0] > G.shape[1]
    if tall:
        G = G.t()
    norm = float(G.norm()) + float(np.float32(eps))
    rows = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else coefficients
    X, s = G, 1 / norm
    f16 = lambda t: (t * 256).half().double() / 256  # noqa: E731

    def times(l, r):  # of two parts each
        return l[0] @ (r[0] + r[1]) + l[1] @ r[0]

    for i, (a, b, c) in enumerate(rows):
        a, b, c = (float(np.float32(v)) for v in (a, b, c))
        if arithmetic == "f16":
            if i == 0:
                e = 2.0 ** -np.floor(np.log2(norm))
                h, lo = _two_parts(X * e, 1024)
                s = s / e
            else:
                h, lo = _two_parts(X, 1024)
                s = 1.0
            A = f16((h @ h.t()) * s * s)
            B = b * A + c * (A @ A)
            diag = torch.diag(B.diagonal())
            X = s * (a * (h + lo) + diag @ (h + lo) + f16(B - diag) @ h)
        else:
            X = X * s if i == 0 else X
            if arithmetic == "two":
                x2 = _two_parts(X, 1024)
                A = times(x2, [v.t() for v in x2])
                a2 = _two_parts(A, 256)
                B = b * (a2[0] + a2[1]) + c * times(a2, a2)
                diag = torch.diag(B.diagonal())
                X = sum(x2)
                X = a * X + diag @ X + times(_two_parts(B - diag, 256), x2)
            else:
                A = X @ X.t()
                X = a * X + (b * A + c * (A @ A)) @ X
    return X.t() if tall else X


def orth_strict(x, steps, coefficients, eps, half):
    """What the steps' roundings may come to at most, to first order, in the Frobenius norm
    (a matrix whose elements are rounded relatively by u is off by u of its norm).  An
    error that reaches a step leaves it at most max |p'| larger, p the step's polynomial
    over the singular values that X has there; each step adds its own:
      A: X's first parts (half: u = 2^-11), a sum of K products, A's rounding;
      B: what A's error makes of b A + c A A, its own sum, its rounding;
      X: B's error, the product with X's first part, its sum, the rounding of the result
    (half: A and B round by 2^-11, X with its second part by 2^-22; not half: two parts, 2^-22,
    and products without that of the second ones, 2^-22 each of both operands.  All have an
    absolute floor, half of float16's last step, 2^-25, over the 2^8 or more that they are
    held times: 2^-33 an element)."""
    G = d64(x)
    if G.shape[0] > G.shape[1]:
        G = G.t()
    p, q = G.shape
    X = G / (float(G.norm()) + float(np.float32(eps)))
    u, ux, ust = (2.0 ** -11, 2.0 ** -11, 2.0 ** -22) if half else (2.0 ** -22,) * 3
    floor = 2.0 ** -33
    e = 4 * E * float(X.norm()) + (floor * np.sqrt(p * q))
    rows = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else coefficients
    for a, b, c in rows:
        top = float(torch.linalg.matrix_norm(X, 2))
        t = torch.linspace(0, 1.01 * top, 4001, dtype=torch.float64)
        grow = float((a + 3 * b * t ** 2 + 5 * c * t ** 4).abs().max())
        A = X @ X.t()
        B = b * A + c * (A @ A)
        nA, nX = float(A.norm()), float(X.norm())
        dA = (2 * ux * nX * top + (q + 4) * E * float((X.abs() @ X.abs().t()).norm()) + u * nA
              + floor * p)
        dB = ((abs(b) + 2 * abs(c) * top ** 2) * dA + u * float(B.norm()) + floor * p
              + (p + 6) * E * float((abs(b) * A.abs() + abs(c) * (A.abs() @ A.abs())).norm()))
        dX = (dB * top + float(B.norm()) * ux * nX
              + (p + 6) * E * float((abs(a) * X.abs() + B.abs() @ X.abs()).norm()))
        X = a * X + B @ X
        e = grow * e + dX + ust * float(X.norm()) + floor * np.sqrt(p * q)
    return e


def check_orth(got, x, steps, coefficients, eps, base=None, scale=1.0, keep=1.0, label=""):
    """In the norm of the result, for each matrix: at most orth_strict's bound.  That is far
    from tight, so from 32 x 32 on (more than a thousand roundings of A and of B, whose norm is
    then near its mean) also twice what the emulated arithmetic is off by: the kernel's
    roundings are the same ones, but fall elsewhere where a float32 sum decides them (K
    roundings of random sign, sqrt(K) E of its terms: beside parts that round by 2^-22 = 4 E
    the sums' share is sqrt(K) / 4).  The result's own rounding, and those of scale and keep, come on top."""
    dt = got.dtype
    half = dt == torch.bfloat16
    xs, gs = (x[None], got[None]) if x.dim() == 2 else (x, got)
    bs = None if base is None else (base[None] if base.dim() == 2 else base)
    for i in range(xs.shape[0]):
        want = orth64(xs[i], steps, coefficients, eps)
        bound = orth_strict(xs[i], steps, coefficients, eps, half)
        if min(want.shape) >= 32:
            model = orth64(xs[i], steps, coefficients, eps, "f16" if half else "two")
            off = float((model - want).norm())
            bound = min(bound, off * (2.0 if half else 2.0 + np.sqrt(max(want.shape)) / 4))
        kept = keep * d64(bs[i]) if bs is not None else torch.zeros_like(want)
        y = scale * want + kept
        bound = (abs(scale) * bound + U[dt] * (float(y.norm()) + abs(scale) * bound)
                 + 3 * E * (abs(scale) * float(want.norm()) + float(kept.norm()))
                 + TINY[dt] * U[dt] * y.numel() ** 0.5)
        far = float((d64(gs[i]) - y).norm())
        assert far <= bound, f"{label} matrix {i}: {far:.3g} off, {bound:.3g} allowed"
