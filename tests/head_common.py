"""64-bit restatements of the hidden-state operators (lsamp_linear,
lsamp_head_loss, lsamp_dropout and their gradients), each with a bound on what
the kernels' arithmetic may be off by.

The bounds are worst cases of the arithmetic that the kernels promise, element
by element: products of `dtype` values summed in float32 (each of K additions
rounds to 2^-24 of the partial sum, at most K 2^-24 sum |a b|), functions
evaluated in float32, the gradient at the pre-activations or logits rounded
once to `dtype`, the result rounded once to its type.  U is a type's unit
roundoff.  Values below a type's normal range round absolutely (TINY).
"""
from __future__ import annotations

import math

import numpy as np
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -14}
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E = 2.0 ** -24


def d64(t):
    return t.detach().cpu().double()


def matrix(rng, rows, cols, dtype, std=1.0, layout="dense"):
    """[rows, cols] on the GPU: "dense", "pad" (rows 8 elements apart more),
    "odd" (a view whose rows start anywhere)."""
    a = torch.from_numpy(rng.standard_normal((rows, cols)) * std).to(dtype)
    if layout == "dense":
        return a.cuda()
    extra, shift = (8, 0) if layout == "pad" else (3, 1)
    wide = torch.full((rows, cols + extra), float("nan"), dtype=dtype, device="cuda")
    wide[:, shift:shift + cols] = a.cuda()
    return wide[:, shift:shift + cols]


def act64(name, z, cap=0.0):
    """act(z), act'(z) in 64 bits."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        s = torch.sigmoid(2 * u)
        return z * s, s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if name == "softcap":
        t = torch.tanh(z / cap)
        return cap * t, 1 - t * t
    return z, torch.ones_like(z)


def sum_bound(k, mags):
    """What a float32 sum of k products may be off by (mags: the sum of their
    magnitudes); one more rounding for a bias."""
    return (k + 2) * E * mags


def linear64(x, w, bias=None, residual=None, act="none", cap=0.0, out_dtype=None):
    out_dtype = out_dtype or x.dtype
    X, Wt = d64(x), d64(w)
    z = X @ Wt.t()
    mags = X.abs() @ Wt.abs().t()
    if bias is not None:
        z, mags = z + d64(bias), mags + d64(bias).abs()
    err = sum_bound(x.shape[1], mags)
    pre, pre_err = z, err
    y, _ = act64(act, z, cap)
    # |act'| <= 1.13 for every activation; its evaluation: 16 roundings of a value at most |z| + 1
    if act != "none":
        err = 1.2 * err + 16 * E * (z.abs() + 1)
    if residual is not None:
        y = y + d64(residual)
        err = err + E * (y.abs() + err)
    return {"out": (y, err + U[out_dtype] * (y.abs() + err) + TINY[out_dtype] * U[out_dtype]),
            "pre": (pre, pre_err)}


def linear_grads64(d_out, x, w, pre, act="none", cap=0.0):
    """From the kernel's own `pre` (float32), as the operator is defined."""
    dt = d_out.dtype
    D, X, Wt = d64(d_out), d64(x), d64(w)
    rows, k, n = x.shape[0], x.shape[1], w.shape[0]
    dz, dz_err = D, torch.zeros_like(D)
    if act != "none":
        z = d64(pre)
        _, slope = act64(act, z, cap)
        dz = D * slope
        dz_err = D.abs() * 24 * E * (z.abs() + 1) + U[dt] * dz.abs() + TINY[dt] * U[dt]
    m = dz.abs() + dz_err

    def product(a, a_err, am, b, count):
        y = a @ b
        err = a_err @ b.abs() + sum_bound(count, am @ b.abs())
        return y, err + U[dt] * (y.abs() + err) + TINY[dt] * U[dt]

    db = dz.sum(0)
    db_err = dz_err.sum(0) + sum_bound(rows, m.sum(0))
    return {"d_x": product(dz, dz_err, m, Wt, n),
            "d_weight": product(dz.t(), dz_err.t(), m.t(), X, rows),
            "d_bias": (db, db_err + U[dt] * (db.abs() + db_err) + TINY[dt] * U[dt])}


def logits64(x, w, bias, cap):
    X, Wt = d64(x), d64(w)
    z = X @ Wt.t()
    mags = X.abs() @ Wt.abs().t()
    if bias is not None:
        b = d64(bias)
        z = z + b
        mags = mags + torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b))
    err = sum_bound(x.shape[1], mags)
    slope = torch.ones_like(z)
    if cap:
        t = torch.tanh(z / cap)
        z, slope = cap * t, 1 - t * t
        err = err + 8 * E * cap
    return z, err, slope


def loss64(x, w, targets, bias=None, cap=0.0):
    z, err, _ = logits64(x, w, bias, cap)
    lse = torch.logsumexp(z, 1)
    t = targets.cpu().long()
    v = w.shape[0]
    ok = (t >= 0) & (t < v)
    zt = z.gather(1, t.clamp(0, v - 1)[:, None])[:, 0]
    loss = torch.where(t < 0, torch.zeros_like(lse),
                       torch.where(ok & ~torch.isneginf(lse), lse - zt,
                                   torch.full_like(lse, float("nan"))))
    # exponentials are relatively off by some roundings of their argument, and
    # the float32 sum by a rounding for each of the levels that add it up
    span = (z.amax(1) - torch.where(torch.isneginf(z), torch.full_like(z, float("inf")), z).amin(1))
    e = err.amax(1) + E * (64 + 2 * span.clamp(min=0).nan_to_num(posinf=0) + 2 * lse.abs().nan_to_num())
    return {"lse": (lse, e), "loss": (loss, 2 * e + 2 * E * zt.abs().nan_to_num())}


def loss_grads64(d_loss, x, w, targets, lse, bias=None, cap=0.0):
    """From the kernel's own `lse` (float32), as the operator is defined."""
    dt = x.dtype
    z, err, slope = logits64(x, w, bias, cap)
    rows, v = x.shape[0], w.shape[0]
    X, Wt = d64(x), d64(w)
    L = d64(lse)
    p = torch.exp(z - L[:, None])
    t = targets.cpu().long()
    ok = (t >= 0) & (t < v) & ~torch.isneginf(L)
    onehot = torch.zeros_like(z)
    onehot[torch.arange(rows), t.clamp(0, v - 1)] = 1
    wt = torch.where(ok, d64(d_loss), torch.zeros_like(L))[:, None]
    dead = ~ok[:, None].expand_as(z)
    g = (wt * (p - onehot) * slope).masked_fill(dead, 0)
    # exp of (z - lse), each rounded; the slope of a cap
    arg = torch.where(torch.isneginf(z), torch.zeros_like(z), z.abs()) + L.abs().nan_to_num()[:, None]
    p_err = p * (err + 4 * E * (arg + 4)) + E
    top = float(d64(d_loss).abs().max()) if rows else 0.0
    small = top * 2.0 ** -39 if dt != torch.float32 else 0.0  # half of float16's last step, unscaled
    g_err = (wt.abs() * p_err * (slope + 8 * E) + 16 * E * g.abs()
             + (U[dt] * g.abs() if dt != torch.float32 else 0) + small).masked_fill(dead, 0)
    m = g.abs() + g_err

    def product(a, a_err, am, b, count):
        y = a @ b
        e = a_err @ b.abs() + sum_bound(count, am @ b.abs())
        return y, e + U[dt] * (y.abs() + e) + TINY[dt] * U[dt]

    db = g.sum(0)
    db_err = g_err.sum(0) + sum_bound(rows, m.sum(0))
    return {"d_x": product(g, g_err, m, Wt, v),
            "d_weight": product(g.t(), g_err.t(), m.t(), X, rows),
            "d_bias": (db, db_err + U[dt] * (db.abs() + db_err) + TINY[dt] * U[dt])}


def philox_keep(rows, cols, p, key, offset):
    """The kept elements of lsamp_dropout, from Philox4x32-10's definition."""
    u64, low = np.uint64, np.uint64(0xFFFFFFFF)
    g = (cols + 7) // 8
    c = [np.tile(np.arange(g, dtype=u64), rows), np.repeat(np.arange(rows, dtype=u64), g),
         np.full(rows * g, offset % 2 ** 32, u64), np.full(rows * g, offset >> 32, u64)]
    k = [key % 2 ** 32, key >> 32]
    for _ in range(10):
        a, b = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
        c = [(b >> u64(32)) ^ c[1] ^ u64(k[0]), b & low, (a >> u64(32)) ^ c[3] ^ u64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.stack([x.astype("<u4") for x in c], 1).view("<u2").reshape(rows, g * 8)[:, :cols]
    return torch.from_numpy(bits >= int(np.rint(np.float64(np.float32(p)) * 65536)))


def check(got, want, label=""):
    """got within want's bound everywhere; NaN where it is NaN, and equal infinities."""
    y, err = want
    g = d64(got)
    assert g.shape == y.shape, f"{label}: {tuple(g.shape)} != {tuple(y.shape)}"
    finite = torch.isfinite(y)
    assert torch.equal(torch.isnan(g), torch.isnan(y)), f"{label}: NaN in other places"
    inf = torch.isinf(y)
    assert torch.equal(g[inf], y[inf]), f"{label}: infinities differ"
    off = (g - y).abs()[finite]
    bound = err[finite]
    bad = ~(off <= bound)
    assert not bad.any(), (f"{label}: {int(bad.sum())} of {bad.numel()} outside the bound, worst "
                           f"{float((off / bound.clamp(min=1e-300)).max()):.3g} times it")
