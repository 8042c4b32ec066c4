"""What the hidden-state operators' functions and scales may be off by, on the GPU
against 64 bits: rows without a loss beside a float16 gradient's scale, soft
caps near and far from saturation, and column sums before rounding."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import head_common as H
import head_sampled as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lsamp.api import Context
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    c = Context(0, max_rows=4, max_vocab=1024)
    yield c
    c.close()


def _inputs(rng, dtype, m, k, v):
    dt = H.DT[dtype]
    x, w = H.matrix(rng, m, k, dt), H.matrix(rng, v, k, dt, 3 / np.sqrt(k))
    t = torch.from_numpy(rng.integers(0, v, m).astype(np.int32)).cuda()
    d = torch.from_numpy(rng.uniform(0.5, 2.0, m).astype(np.float32)).cuda() / m
    return x, w, t, d


# ---------------------------------------------------- the scale of a 16-bit gradient
@pytest.mark.parametrize("value", [1e6, float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_rows_without_a_loss_set_no_scale(ctx, dtype, value):
    """What d_loss holds at ignored rows, at targets out of range and at rows with
    no logit changes no bit of the gradients."""
    m, k, v = 70, 64, 900
    rng = np.random.default_rng(31)
    x, w, t, d = _inputs(rng, dtype, m, k, v)
    w[:, 0] = w[:, 0].abs() + 0.1
    x[20] = 0
    x[20, 0] = float("-inf")  # (every logit -inf)
    t[5], t[6], t[7] = -100, v, 2 ** 31 - 1
    f = ctx.prepare_head_loss(x, w, t)
    f.launch()
    assert torch.isneginf(f.lse[20])
    x[20, 0] = 0  # (0 x -inf is no number, in d_weight)
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, want_bias=True)
    p.launch()
    clean = {n: g.clone() for n, g in p.outputs().items()}
    want = S.head_grads(d, x, w, t, f.lse, None, 0.0)
    for n, g in clean.items():
        H.check(g, want[n], n)
    d[[5, 6, 7, 20]] = value
    p.launch()
    for n, g in p.outputs().items():
        assert torch.equal(g, clean[n]), n


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_an_infinite_gradient_stays_in_its_row(ctx, dtype):
    """A row whose d_loss is no finite number sets no scale: the rows beside it have
    the d_x that they have without it."""
    m, k, v = 70, 64, 900
    rng = np.random.default_rng(32)
    x, w, t, d = _inputs(rng, dtype, m, k, v)
    f = ctx.prepare_head_loss(x, w, t)
    f.launch()
    ignored = t.clone()
    ignored[[9, 40]] = -1
    want = ctx.prepare_head_loss_backward(d, x, w, ignored, lse=f.lse, want_weight=False)
    want.launch()
    d[9], d[40] = float("inf"), float("nan")
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, want_weight=False)
    p.launch()
    rest = torch.ones(m, dtype=torch.bool)
    rest[[9, 40]] = False
    assert torch.equal(p.d_x[rest.cuda()], want.d_x[rest.cuda()])
    assert not torch.isfinite(p.d_x[[9, 40]].float()).any()


# ------------------------------------------------------------------------- soft caps
def _capped(dtype, cap):
    """One row of one feature: the logits are the weights themselves, t = z / cap
    from -12 to 12, and the target another id."""
    dt = H.DT[dtype]
    z = (torch.linspace(-12, 12, 385) * cap).to(dt)
    w = torch.cat([z, z[:1] * 0])[:, None].cuda()
    return torch.ones(1, 1, dtype=dt, device="cuda"), w, torch.tensor([385], dtype=torch.int32).cuda()


@pytest.mark.parametrize("cap", [0.5, 30.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_slope_of_a_capped_logit(ctx, dtype, cap):
    """softcap' = 4 e / (1 + e)^2, e = exp(-2 |t|), is relatively right at both signs,
    down to 1e-10 at t = -12 as at 12."""
    x, w, t = _capped(dtype, cap)
    d = torch.ones(1, device="cuda")
    f = ctx.prepare_head_loss(x, w, t, softcap=cap)
    f.launch()
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, softcap=cap, want_bias=True)
    p.launch()
    want = S.head_grads(d, x, w, t, f.lse, None, cap)
    for n, g in p.outputs().items():
        H.check(g, want[n], n)
    y, err = want["d_weight"]
    if dtype != "f16":  # (float16 holds no 1e-10)
        assert float((err / y.abs())[:385].max()) < 2.0 ** -6, "the bound has become empty"


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_slope_of_a_capped_activation(ctx, dtype):
    """The same of a linear block whose activation is a soft cap, from `pre`."""
    cap = 5.0
    pre = (torch.linspace(-12, 12, 385) * cap)[None, :].cuda()
    dt = H.DT[dtype]
    one = torch.ones(1, 385, dtype=dt, device="cuda")
    p = ctx.prepare_linear_backward(one, one[:, :1], one.t().contiguous(), pre=pre,
                                    activation="softcap", softcap=cap, want_x=False, want_bias=True)
    p.launch()
    t = H.d64(pre)[0] / cap
    e = torch.exp(-2 * t.abs())
    y = 4 * e / (1 + e) ** 2
    want = S.rounded(y, y * H.E * (16 + 8 * t.abs()), dt)
    H.check(p.d_bias, want, "d_bias")
    H.check(p.d_weight[:, 0], want, "d_weight")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_small_logits_under_a_large_cap(ctx, dtype):
    """cap tanh(z / cap) of logits far below the cap is as near as the logits' own
    sums: a cap of 10^4 or 10^6 loses nothing."""
    m, k, v = 40, 64, 900
    rng = np.random.default_rng(33)
    x, w, t, d = _inputs(rng, dtype, m, k, v)
    X, W = H.d64(x), H.d64(w)
    raw = X @ W.t()
    for cap in (1e4, 1e6, 1e38):
        f = ctx.prepare_head_loss(x, w, t, softcap=cap)
        f.launch()
        z = cap * torch.tanh(raw / cap)
        err = (H.sum_bound(k, X.abs() @ W.abs().t()) + 16 * H.E * z.abs()).amax(1)
        lse = torch.logsumexp(z, 1)
        zt = z.gather(1, t.cpu().long()[:, None])[:, 0]
        e = err + H.E * (64 + 2 * (z.amax(1) - z.amin(1)) + 2 * lse.abs())
        H.check(f.lse, (lse, e), f"lse, cap {cap:g}")
        H.check(f.loss, (lse - zt, 2 * e + 2 * H.E * zt.abs()), f"loss, cap {cap:g}")


def test_small_float32_gradients_keep_their_bits(ctx):
    """A loss times a power of two has its gradients times that power, bit for bit,
    as long as they are normal numbers: also where bfloat16 parts of the gradient
    at the logits would not be."""
    m, k, v = 200, 64, 900
    rng = np.random.default_rng(35)
    x, w, t, d = _inputs(rng, "f32", m, k, v)
    f = ctx.prepare_head_loss(x, w, t)
    f.launch()
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, want_bias=True)
    p.launch()
    one = {n: g.clone() for n, g in p.outputs().items()}
    for e in (-106, -60, 60, 110):
        d.mul_(2.0 ** e)
        p.launch()
        d.mul_(2.0 ** -e)
        for n, g in p.outputs().items():
            normal = one[n].abs() > 2.0 ** -18
            assert normal.any()
            assert torch.equal(g[normal] * 2.0 ** -e, one[n][normal]), (n, e)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_bias_of_minus_infinity_under_a_cap(ctx, dtype):
    """A capped logit is at least -softcap, also where the bias is -inf: the id keeps
    that mass, and has no gradient."""
    m, k, v, cap = 70, 64, 900, 2.0
    rng = np.random.default_rng(34)
    x, w, t, d = _inputs(rng, dtype, m, k, v)
    b = H.matrix(rng, 1, v, H.DT[dtype], 0.5)[0]
    b[::3] = float("-inf")
    f = ctx.prepare_head_loss(x, w, t, bias=b, softcap=cap)
    f.launch()
    want = H.loss64(x, w, t, b, cap)
    H.check(f.lse, want["lse"], "lse")
    H.check(f.loss, want["loss"], "loss")
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, bias=b, softcap=cap, want_bias=True)
    p.launch()
    want = S.head_grads(d, x, w, t, f.lse, b, cap)
    for n, g in p.outputs().items():
        H.check(g, want[n], n)
    assert (p.d_weight[::3] == 0).all()


# ------------------------------------------------------------------------ column sums
@pytest.mark.parametrize("m,v,layout", [(1, 300, "dense"), (40, 1003, "dense"), (64, 777, "odd"),
                                        (300, 2100, "dense"), (1100, 5000, "dense"),
                                        (300, 1999, "odd"), (2050, 70001, "dense"),
                                        (20011, 333, "dense")])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_head_bias_gradient_sums_in_float32(ctx, dtype, m, v, layout):
    """d_bias adds up the gradient at the logits before it is rounded for the products."""
    rng = np.random.default_rng(m + v)
    k = 72
    dt = H.DT[dtype]
    x, w = H.matrix(rng, m, k, dt, layout=layout), H.matrix(rng, v, k, dt, 3 / np.sqrt(k), layout)
    # (few targets: their columns' sums nearly cancel against their probabilities)
    t = torch.from_numpy(rng.integers(0, min(v, 20), m).astype(np.int32)).cuda()
    d = torch.from_numpy(rng.uniform(0.5, 2.0, m).astype(np.float32)).cuda() / m
    f = ctx.prepare_head_loss(x, w, t)
    f.launch()
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, want_bias=True)
    p.launch()
    ids = S.sample(rng, v, 100, *range(min(v, 20)))
    c, own, _ = S.loss_grad(d, x, w[ids.cuda()], t, f.lse, None, 0.0, ids, 0.0)
    err = own.sum(0) + H.sum_bound(m, (c.abs() + own).sum(0))
    H.check(p.d_bias[ids.cuda()], S.rounded(c.sum(0), err, dt), "d_bias")
    only = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, want_x=False, want_weight=False,
                                          want_bias=True)
    only.launch()
    assert torch.equal(only.d_bias, p.d_bias)
