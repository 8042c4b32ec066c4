"""Large results of the hidden-state operators in 64 bits, whole or at sampled rows
and columns, with bounds derived as in head_common.py.  The 64-bit products run
where their inputs are.  A row of d_x needs its own row of x and all of the weight,
a row of d_weight its own row of the weight and all of x."""
from __future__ import annotations

import torch

import head_common as H


def sample(rng, n, count, *also):
    """Some of 0 .. n - 1: both ends, both sides of multiples of 256, `also`,
    and others at random."""
    at = {0, n - 1, *[i for i in (63, 64, 127, 128, 255, 256, n // 256 * 256 - 1, n // 256 * 256)
                      if 0 <= i < n], *[int(i) for i in also]}
    at |= {int(i) for i in rng.integers(0, n, count)}
    return torch.tensor(sorted(at))


def d64(t):
    return t.detach().double()


def rounded(y, err, dt):
    """(y, err) with the rounding to `dt`, on the CPU."""
    return y.cpu(), (err + H.U[dt] * (y.abs() + err) + H.TINY[dt] * H.U[dt]).cpu()


def product(a, a_err, b, count, dt):
    y = a @ b
    return rounded(y, a_err @ b.abs() + H.sum_bound(count, (a.abs() + a_err) @ b.abs()), dt)


def linear(x, w, bias, residual, act, cap, out_dtype):
    """out and pre of a linear block."""
    X, W = d64(x), d64(w)
    z, mags = X @ W.t(), X.abs() @ W.abs().t()
    if bias is not None:
        z, mags = z + d64(bias), mags + d64(bias).abs()
    err = H.sum_bound(x.shape[1], mags)
    y, _ = H.act64(act, z, cap)
    pre = (z.cpu(), err.cpu())
    if act != "none":
        err = 1.2 * err + 16 * H.E * (z.abs() + 1)
    if residual is not None:
        y = y + d64(residual)
        err = err + H.E * (y.abs() + err)
    return {"out": rounded(y, err, out_dtype), "pre": pre}


def linear_grads(d_out, x, w, pre, act, cap, rows=None, outs=None):
    """d_x (at `rows`), d_weight and d_bias (at the outputs `outs`)."""
    dt, dev = d_out.dtype, d_out.device
    X, W = d64(x), d64(w)

    def dz(sl):
        D = d64(d_out[sl])
        if act == "none":
            return D, torch.zeros_like(D), torch.zeros_like(D)
        z = d64(pre[sl])
        y = D * H.act64(act, z, cap)[1]
        own = D.abs() * 24 * H.E * (z.abs() + 1)  # of the slope, in float32
        return y, own, own + H.U[dt] * y.abs() + H.TINY[dt] * H.U[dt]

    r, _, r_err = dz(slice(None) if rows is None else rows.to(dev))
    o, o_own, o_err = dz((slice(None), slice(None) if outs is None else outs.to(dev)))
    db_err = o_own.sum(0) + H.sum_bound(x.shape[0], (o.abs() + o_own).sum(0))
    return {"d_x": product(r, r_err, W, w.shape[0], dt),
            "d_weight": product(o.t(), o_err.t(), X, x.shape[0], dt),
            "d_bias": rounded(o.sum(0), db_err, dt)}


def logits(x, w, bias, cap):
    """Logits, their error, the cap's slope and its relative error."""
    X, W = d64(x), d64(w)
    z, mags = X @ W.t(), X.abs() @ W.abs().t()
    if bias is not None:
        b = d64(bias)
        z, mags = z + b, mags + b.abs().masked_fill(torch.isinf(b), 0)
    err = H.sum_bound(x.shape[1], mags)
    slope, slope_rel = torch.ones_like(z), torch.zeros_like(z)
    if cap:
        t = z / cap
        e = torch.exp(-2 * t.abs())
        # (relatively: twice the argument's own error, and some roundings of a function)
        slope, slope_rel = 4 * e / (1 + e) ** 2, 4 * err / cap + H.E * (16 + 8 * t.abs())
        slope_rel = slope_rel.nan_to_num(posinf=0)  # (a slope of 0)
        z, err = cap * torch.tanh(t), err + 8 * H.E * cap
    return z, err, slope, slope_rel


def loss(x, w, targets, bias, cap):
    """lse and loss of rows whose targets are in range or negative."""
    z, err, _, _ = logits(x, w, bias, cap)
    lse = torch.logsumexp(z, 1)
    t = targets.long()
    zt = z.gather(1, t.clamp(min=0)[:, None])[:, 0]
    span = z.amax(1) - z.masked_fill(torch.isinf(z), float("inf")).amin(1)
    e = err.amax(1) + H.E * (64 + 2 * span + 2 * lse.abs())
    y = torch.where(t < 0, torch.zeros_like(lse), lse - zt)
    return {"lse": (lse.cpu(), e.cpu()), "loss": (y.cpu(), (2 * e + 2 * H.E * zt.abs()).cpu())}


def loss_grad(d_loss, x, w, targets, lse, bias, cap, ids, top):
    """The gradient at the logits of the ids `ids` (whose rows `w` holds), and what
    it may be off by in float32 and as it is stored.  `top`: the largest |d_loss| of
    a row with a loss, which the scale of a 16-bit gradient goes by."""
    dt, dev = x.dtype, x.device
    z, err, slope, slope_rel = logits(x, w, bias, cap)
    L = d64(lse)[:, None]
    t = targets.to(dev).long()
    ok = (t >= 0) & ~torch.isneginf(L[:, 0])
    onehot = (t[:, None] == ids.to(dev)[None, :]).double()
    p = torch.exp(z - L)
    wt = torch.where(ok, d64(d_loss), torch.zeros_like(L[:, 0]))[:, None]
    dead = ~ok[:, None].expand_as(z)
    g = (wt * (p - onehot) * slope).masked_fill(dead, 0)
    arg = z.abs().masked_fill(torch.isinf(z), 0) + L.abs().nan_to_num()
    p_err = p * (err + 4 * H.E * (arg + 4)) + H.E * onehot  # (the target's difference, rounded)
    own = (wt.abs() * p_err * slope + g.abs() * (16 * H.E + slope_rel)).masked_fill(dead, 0)
    stored = own
    if dt != torch.float32:  # rounded once
        stored = own + H.U[dt] * g.abs()
    if dt == torch.float16:  # half of its last step, unscaled
        stored = stored + (top * 2.0 ** -39 * ok.double())[:, None]
    return g, own, stored


def head_grads(d_loss, x, w, targets, lse, bias, cap, rows=None, ids=None):
    """d_x (at `rows`), d_weight and d_bias (at the ids `ids`), from the kernel's own
    lse.  d_bias sums the gradient before it is rounded."""
    dt, dev = x.dtype, x.device
    every = torch.arange(w.shape[0])
    rows, ids = torch.arange(x.shape[0]) if rows is None else rows, every if ids is None else ids
    t = targets.to(dev).long()
    live = (t >= 0) & (t < w.shape[0]) & ~torch.isneginf(lse)
    t = torch.where(live, t, torch.full_like(t, -1))
    d = d64(d_loss)[live].abs()
    d = d[torch.isfinite(d)]
    top = float(d.max()) if len(d) else 0.0
    ri, ci = rows.to(dev), ids.to(dev)
    r, _, r_err = loss_grad(d_loss[ri], x[ri], w, t[ri], lse[ri], bias, cap, every, top)
    d_x = product(r, r_err, d64(w), w.shape[0], dt)
    del r, r_err
    c, c_own, c_err = loss_grad(d_loss, x, w[ci], t, lse, None if bias is None else bias[ci], cap,
                                ids, top)
    db_err = c_own.sum(0) + H.sum_bound(x.shape[0], (c.abs() + c_own).sum(0))
    return {"d_x": d_x, "d_weight": product(c.t(), c_err.t(), d64(x), x.shape[0], dt),
            "d_bias": rounded(c.sum(0), db_err, dt)}
