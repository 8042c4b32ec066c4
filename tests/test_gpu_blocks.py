"""Layer norm, its gradients, rows of 8-bit integers and their products, and
orthogonalised updates on the GPU against 64-bit restatements
(blocks_common.py): one row to thousands, odd sizes, any alignment and stride,
NaN and infinities, streams, graphs, and refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import blocks_common as B
import head_common as H
from lsamp import _ffi

pytestmark = pytest.mark.gpu
MUON = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def ctx():
    from lsamp.api import Context
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    c = Context(0, max_rows=4, max_vocab=1024)
    yield c
    c.close()


# ----------------------------------------------------------------- layer norm
NORM = [
    # rows, cols, weight, bias, residual, layout
    (1, 1, True, True, True, "dense"),
    (1, 2048, True, True, False, "dense"),
    (3, 7, True, False, True, "odd"),
    (5, 513, False, True, False, "odd"),
    (130, 64, True, True, True, "pad"),
    (67, 2049, True, True, True, "dense"),
    (40, 4096, False, False, True, "dense"),
    (9, 4104, True, True, False, "pad"),
    (7, 16384, True, True, True, "dense"),
    (6, 16385, True, True, True, "odd"),
    (70, 20000, True, True, True, "dense"),
    (1030, 200, True, True, True, "dense"),   # (a wave a row)
    (1025, 1000, True, False, False, "odd"),
    (2100, 1999, True, True, True, "pad"),
    (3000, 8, True, True, False, "dense"),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", NORM, ids=lambda c: "-".join(map(str, c)))
def test_layer_norm(ctx, case, dtype):
    rows, n, has_w, has_b, has_r, layout = case
    print(f"norm {case} {dtype}", flush=True)
    rng = np.random.default_rng(rows * 1000003 + n)
    dt = H.DT[dtype]
    x = H.matrix(rng, rows, n, dt, layout=layout)
    x += torch.from_numpy(rng.standard_normal((rows, 1)) * 2).to(dt).cuda()
    w = H.matrix(rng, 1, n, dt)[0] if has_w else None
    b = H.matrix(rng, 1, n, dt)[0] if has_b else None
    d = H.matrix(rng, rows, n, dt, layout=layout)
    res = H.matrix(rng, rows, n, dt, layout=layout) if has_r else None
    wide = torch.full((rows, n + 5), 7.0, dtype=dt, device="cuda")
    p = ctx.prepare_layer_norm(x, weight=w, bias=b, eps=1e-5, want_stats=True, out=wide[:, 2:2 + n])
    p.launch()
    want = B.norm64(x, w, b, 1e-5)
    H.check(p.out, want["out"], "out")
    H.check(p.mean, want["mean"], "mean")
    H.check(p.rstd, want["rstd"], "rstd")
    assert (wide[:, :2] == 7).all() and (wide[:, 2 + n:] == 7).all()
    assert torch.equal(ctx.layer_norm(x, weight=w, bias=b, eps=1e-5), p.out)
    kw = dict(mean=p.mean, rstd=p.rstd, weight=w, residual=res, want_bias=True)
    q = ctx.prepare_layer_norm_backward(d, x, **kw)
    q.launch()
    first = {k: v.clone() for k, v in q.outputs().items()}
    q.launch()
    want = B.norm_grads64(d, x, p.mean, p.rstd, w, res)
    for name, g in q.outputs().items():
        H.check(g, want[name], name)
        assert torch.equal(first[name], g), f"two launches differ in {name}"
    # each gradient alone is the same
    alone = ctx.prepare_layer_norm_backward(d, x, **dict(kw, want_weight=False, want_bias=False))
    alone.launch()
    assert torch.equal(alone.d_x, q.d_x)
    sums = ctx.prepare_layer_norm_backward(d, x, **dict(kw, want_x=False, residual=None))
    sums.launch()
    assert torch.equal(sums.d_weight, q.d_weight) and torch.equal(sums.d_bias, q.d_bias)
    assert set(sums.outputs()) == {"d_weight", "d_bias"}


def test_layer_norm_of_equal_values(ctx):
    """No variance: out is the bias, whatever the offset; gradients are finite."""
    x = torch.full((3, 300), 1000.0, device="cuda")
    x[1] = 0.0
    b = torch.randn(300, device="cuda")
    p = ctx.prepare_layer_norm(x, bias=b, want_stats=True)
    p.launch()
    H.check(p.out, B.norm64(x, None, b, 1e-5)["out"])
    d = torch.randn((3, 300), device="cuda")
    q = ctx.prepare_layer_norm_backward(d, x, mean=p.mean, rstd=p.rstd, want_bias=True)
    q.launch()
    assert all(torch.isfinite(v).all() for v in q.outputs().values())


@pytest.mark.parametrize("rows,n", [(5, 600), (1100, 600), (4, 17000)])
def test_layer_norm_nan_and_infinity_stay_in_their_rows(ctx, rows, n):
    rng = np.random.default_rng(n)
    x = H.matrix(rng, rows, n, torch.bfloat16)
    y = ctx.layer_norm(x)
    z = x.clone()
    z[1, 3], z[3, n - 1] = float("nan"), float("inf")
    got = ctx.layer_norm(z)
    assert torch.isnan(got[1]).all() and torch.isnan(got[3]).all()
    keep = [r for r in range(rows) if r not in (1, 3)]
    assert torch.equal(got[keep], y[keep])


@pytest.mark.parametrize("rows,n", [(50, 777), (600, 4000), (1200, 300), (20, 9000), (40, 17000)])
def test_layer_norm_in_place(ctx, rows, n):
    rng = np.random.default_rng(8)
    x, r = (H.matrix(rng, rows, n, torch.float16) for _ in range(2))
    p = ctx.prepare_layer_norm(x, want_stats=True)
    p.launch()
    d = p.out.clone()
    q = ctx.prepare_layer_norm_backward(d, x, mean=p.mean, rstd=p.rstd, residual=r)
    q.launch()
    into = r.clone()
    ctx.prepare_layer_norm_backward(d, x, mean=p.mean, rstd=p.rstd, residual=into, d_x=into).launch()
    assert torch.equal(into, q.d_x)
    into = d.clone()
    s = ctx.prepare_layer_norm_backward(into, x, mean=p.mean, rstd=p.rstd, residual=r, d_x=into)
    s.launch()
    assert torch.equal(into, q.d_x)
    H.check(s.d_weight, B.norm_grads64(d, x, p.mean, p.rstd, None, r)["d_weight"])
    z = x.clone()
    ctx.layer_norm(z, out=z)
    assert torch.equal(z, p.out)


def test_layer_norm_gradient_against_differences(ctx):
    """float32: the slope of sum(d y) along a direction u, from two forward passes 2 h apart.
    The third derivative's share is h^2 / 6 of a size like the slope's; y rounds to E of
    its few units, n of them, over 2 h."""
    rng = np.random.default_rng(2)
    rows, n, h = 6, 64, 1e-2
    x, d, u = (H.matrix(rng, rows, n, torch.float32) for _ in range(3))
    w, b, uw = (H.matrix(rng, 1, n, torch.float32)[0] for _ in range(3))
    p = ctx.prepare_layer_norm(x, weight=w, bias=b, want_stats=True)
    p.launch()
    q = ctx.prepare_layer_norm_backward(d, x, mean=p.mean, rstd=p.rstd, weight=w, want_bias=True)
    q.launch()
    D = H.d64(d)

    def f(s):
        return float((H.d64(ctx.layer_norm((x.double() + s * u.double()).float(),
                                           weight=(w.double() + s * uw.double()).float(),
                                           bias=b)) * D).sum())
    slope = (f(h) - f(-h)) / (2 * h)
    told = float((H.d64(q.d_x) * H.d64(u)).sum() + (H.d64(q.d_weight) * H.d64(uw)).sum())
    size = float((H.d64(q.d_x).abs() * H.d64(u).abs()).sum())
    noise = 16 * H.E * float((D.abs() * 4).sum()) / (2 * h)
    assert abs(slope - told) <= 20 * h * h * size + noise


# ------------------------------------------------------------ 8-bit integers
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,n,layout", [
    (1, 1, "dense"), (1, 2048, "dense"), (3, 15, "odd"), (64, 4096, "dense"), (5, 513, "odd"),
    (1100, 300, "pad"), (1030, 2047, "odd"), (4, 16384, "dense"), (3, 16399, "odd"),
    (2, 40000, "dense")])
def test_quantize_rows(ctx, rows, n, layout, dtype):
    print(f"quantize {rows} {n} {layout} {dtype}", flush=True)
    rng = np.random.default_rng(rows * 7919 + n)
    x = H.matrix(rng, rows, n, H.DT[dtype], layout=layout)
    wide = torch.full((rows, n + 5), 99, dtype=torch.int8, device="cuda")
    p = ctx.prepare_quantize_rows(x, q=wide[:, 3:3 + n])
    p.launch()
    q, scale = B.quantize64(x)
    assert torch.equal(p.q.cpu(), q) and torch.equal(p.scale.cpu(), scale)
    assert (wide[:, :3] == 99).all() and (wide[:, 3 + n:] == 99).all()


def test_quantize_rows_borders(ctx):
    """Ties, rows of zeros, the smallest and largest numbers, NaN and infinities."""
    x = torch.zeros((12, 260))
    x[0, :254] = torch.arange(-127, 127) + 0.5   # ties of scale 1
    x[0, 255] = 127.0
    x[2] = 2.0 ** -149
    x[3] = torch.linspace(-1, 1, 260) * 2.0 ** -120
    x[4] = torch.linspace(-1, 1, 260) * 3.4e38
    x[5, 7] = float("nan")
    x[6, 9] = float("inf")
    x[7, 259] = -float("inf")
    x[8] = torch.linspace(-1, 1, 260) * 2.0 ** -140
    g = torch.Generator().manual_seed(1)
    x[9] = (torch.randint(-127, 127, (260,), generator=g) + 0.5) * 2.0 ** -7  # (scale beside a power of two)
    x[10] = torch.randn(260, generator=g)
    x[11] = -0.0
    q, scale = ctx.quantize_rows(x.cuda())
    want_q, want_scale = B.quantize64(x)
    assert torch.equal(q.cpu(), want_q)
    assert torch.equal(scale.cpu().nan_to_num(7.0), want_scale.nan_to_num(7.0))
    assert torch.isnan(scale[5:8]).all() and not torch.isnan(scale[:5]).any()


INT8 = [
    # rows, in, out, activation, bias, residual, layout
    (1, 1, 1, "none", False, False, "dense"),
    (1, 7, 5, "relu", True, True, "odd"),
    (1, 2048, 300, "silu", True, True, "dense"),
    (2, 64, 64, "gelu", True, False, "pad"),
    (5, 136, 67, "gelu_tanh", False, True, "dense"),
    (16, 320, 129, "softcap", True, True, "pad"),
    (17, 65, 130, "silu", True, True, "odd"),
    (33, 1000, 96, "none", True, False, "dense"),
    (64, 200, 16390, "relu", False, True, "dense"),
    (64, 130, 257, "relu", False, True, "odd"),
    (65, 512, 64, "gelu", True, True, "pad"),
    (100, 33, 1029, "softcap", True, False, "dense"),
    (129, 200, 257, "gelu_tanh", True, True, "odd"),
    (300, 1040, 520, "silu", False, False, "dense"),
    (515, 72, 264, "none", True, True, "dense"),
    (70, 8208, 72, "gelu", True, True, "dense"),   # (the reduction in parts)
    (70, 8209, 72, "gelu", True, True, "odd"),
    (2100, 160, 2100, "none", True, True, "dense"),
    (2051, 2049, 2053, "silu", True, True, "dense"),
    (2, 1001, 200, "gelu", True, True, "odd"),       # (quantised by every work-group)
    (2, 4096, 16, "none", True, False, "dense"),
    (4, 1100, 16, "none", True, False, "dense"),
    (1, 8192, 40, "none", True, False, "dense"),
    (1, 100, 65700, "silu", True, True, "odd"),      # (a wave's own columns)
    (9, 300, 65601, "none", True, False, "pad"),
    (13, 1500, 32801, "silu", True, True, "odd"),    # (lines of eight waves' columns)
    (17, 260, 33000, "relu", True, True, "dense"),
    (64, 130, 40003, "none", False, True, "odd"),
    (64, 2100, 300, "none", True, True, "odd"),      # (too long to be kept)
    (40, 5000, 130, "silu", True, False, "dense"),
    (16, 9000, 70, "none", False, False, "odd"),
    (50, 3100, 16400, "none", True, True, "dense"),
]


def _quantized(rng, rows, cols, layout):
    a = torch.from_numpy(rng.integers(-127, 128, (rows, cols))).to(torch.int8)
    s = torch.from_numpy(rng.uniform(0.5, 1.5, rows) / 127 / np.sqrt(cols)).float().cuda()
    if layout == "dense":
        return a.cuda(), s
    extra, shift = (16, 0) if layout == "pad" else (3, 1)
    wide = torch.full((rows, cols + extra), 55, dtype=torch.int8, device="cuda")
    wide[:, shift:shift + cols] = a.cuda()
    return wide[:, shift:shift + cols], s


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", INT8, ids=lambda c: "-".join(map(str, c)))
def test_linear_int8(ctx, case, dtype):
    rows, k, n, act, bias, residual, layout = case
    print(f"int8 {case} {dtype}", flush=True)
    rng = np.random.default_rng(rows * 1000003 + k * 1009 + n)
    dt = H.DT[dtype]
    x = H.matrix(rng, rows, k, dt, layout=layout)
    w, ws = _quantized(rng, n, k, layout)
    b = H.matrix(rng, 1, n, dt)[0] if bias else None
    res = H.matrix(rng, rows, n, dt, layout=layout) if residual else None
    kw = dict(bias=b, residual=res, activation=act, softcap=5.0)
    p = ctx.prepare_linear_int8(x, w, ws, **kw)
    p.launch()
    q, xs = B.quantize64(x)
    H.check(p.out, B.int8_64(q, xs, w, ws, b, res, act, 5.0, dt), "out")
    first = p.out.clone()
    p.launch()
    assert torch.equal(first, p.out), "two launches differ"
    # quantised by the caller: the same bits, also from rows of any alignment
    gq, gs = ctx.quantize_rows(x)
    assert torch.equal(ctx.linear_int8(gq, w, ws, x_scale=gs, out_dtype=dt, **kw), first)
    odd = torch.full((rows, k + 3), 9, dtype=torch.int8, device="cuda")[:, 1:1 + k]
    odd.copy_(gq)
    assert torch.equal(ctx.linear_int8(odd, w, ws, x_scale=gs, out_dtype=dt, **kw), first)
    # into padded buffers whose rest is left alone; float32 out
    into = torch.full((rows, n + 5), 7.0, dtype=dt, device="cuda")
    ctx.linear_int8(x, w, ws, out=into[:, 3:3 + n], **kw)
    assert torch.equal(into[:, 3:3 + n], first)
    assert (into[:, :3] == 7).all() and (into[:, 3 + n:] == 7).all()
    wide = torch.full((rows, n + 5), 7.0, device="cuda")
    ctx.linear_int8(x, w, ws, out=wide[:, 2:2 + n], **kw)
    H.check(wide[:, 2:2 + n], B.int8_64(q, xs, w, ws, b, res, act, 5.0, dt, torch.float32), "float32")
    assert (wide[:, :2] == 7).all() and (wide[:, 2 + n:] == 7).all()


def test_linear_int8_largest_sums(ctx):
    """Whole sums next to 2^31 (-128 times -128, which a caller's own weights may hold)."""
    k = 131071
    for rows in (1, 70):
        q = torch.full((rows, k), -128, dtype=torch.int8, device="cuda")
        w = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
        w[1] = 127
        w[2, ::2] = 127
        one = torch.ones(rows, device="cuda")
        got = ctx.linear_int8(q, w, torch.ones(3, device="cuda"), x_scale=one, out_dtype=torch.float32)
        want = (q[0].cpu().long() * w.cpu().long()).sum(1)
        assert torch.equal(got[0].cpu(), want.float()) and torch.equal(got[-1], got[0])


@pytest.mark.parametrize("rows", [4, 40, 200])
def test_linear_int8_nan_stays_in_its_row(ctx, rows):
    rng = np.random.default_rng(rows)
    x = H.matrix(rng, rows, 192, torch.bfloat16)
    w, ws = _quantized(rng, 96, 192, "dense")
    y = ctx.linear_int8(x, w, ws)
    z = x.clone()
    z[1, 3], z[3, 0] = float("nan"), -float("inf")
    z[2] = 0
    got = ctx.linear_int8(z, w, ws)
    assert torch.isnan(got[1]).all() and torch.isnan(got[3]).all() and (got[2] == 0).all()
    keep = [r for r in range(rows) if r not in (1, 2, 3)]
    assert torch.equal(got[keep], y[keep])


def test_linear_int8_follows_linear(ctx):
    """The quantised block beside the block it stands for: each operand is off by at most
    half a step of its row's scale, so a sum by at most that of either side."""
    rng = np.random.default_rng(4)
    x, w = H.matrix(rng, 70, 384, torch.float32), H.matrix(rng, 100, 384, torch.float32, 0.05)
    q, s = ctx.quantize_rows(w)
    off = H.d64(ctx.linear_int8(x, q, s)) - H.d64(ctx.linear(x, w))
    hx, hw = H.d64(x).abs().amax(1) / 254, H.d64(w).abs().amax(1) / 254
    bound = (hx[:, None] * H.d64(w).abs().sum(1) + hw * H.d64(x).abs().sum(1)[:, None]
             + 384 * hx[:, None] * hw)
    assert (off.abs() <= 1.001 * bound).all()


@pytest.mark.parametrize("rows,k,n", [(40, 96, 96), (1, 96, 300), (20, 600, 33000), (300, 64, 700),
                                      (2000, 300, 2000)])
def test_linear_int8_residual_in_place(ctx, rows, k, n):
    rng = np.random.default_rng(5)
    x, r = H.matrix(rng, rows, k, torch.bfloat16), H.matrix(rng, rows, n, torch.bfloat16)
    w, ws = _quantized(rng, n, k, "dense")
    y = ctx.linear_int8(x, w, ws, activation="silu", residual=r)
    z = r.clone()
    ctx.linear_int8(x, w, ws, activation="silu", residual=z, out=z)
    assert torch.equal(y, z)


# ----------------------------------------------------- orthogonalised updates
def _momentum(rng, batch, m, n, dtype, layout="dense", size=1e-3):
    """A falling spectrum above noise; many singular values are small."""
    r = max(1, min(m, n) // 2)
    fall = 1 / (np.arange(r) + 3.0)
    a = np.stack([(rng.standard_normal((m, r)) * fall) @ rng.standard_normal((r, n))
                  + 0.02 * rng.standard_normal((m, n)) for _ in range(batch)]) * size
    t = torch.from_numpy(a).to(dtype)
    if layout == "dense":
        return t.cuda()
    wide = torch.full((batch, m + 1, n + 3), float("nan"), dtype=dtype, device="cuda")
    wide[:, :m, 1:1 + n] = t.cuda()
    return wide[:, :m, 1:1 + n]


ORTH = [
    # batch, rows, cols, steps, layout
    (1, 1, 1, 5, "dense"),
    (1, 1, 300, 3, "dense"),
    (2, 9, 5, 5, "odd"),
    (1, 64, 64, 5, "dense"),
    (3, 63, 65, 5, "odd"),
    (1, 130, 70, 5, "dense"),
    (2, 72, 200, 6, "odd"),
    (4, 256, 256, 5, "dense"),
    (1, 333, 500, 5, "odd"),
    (1, 520, 264, 5, "dense"),
    (1, 1000, 1100, 2, "dense"),
    (1, 7, 5000, 5, "odd"),
    (1, 5000, 7, 5, "odd"),
]


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32"), ("f16", "f16"),
                                   ("bf16", "f32")], ids="-".join)
@pytest.mark.parametrize("case", ORTH, ids=lambda c: "-".join(map(str, c)))
def test_orthogonalize(ctx, case, types):
    batch, m, n, steps, layout = case
    print(f"orth {case} {types}", flush=True)
    rng = np.random.default_rng(m * 1000003 + n * 101 + steps)
    x = _momentum(rng, batch, m, n, H.DT[types[0]], layout)
    dt = H.DT[types[1]]
    got = ctx.orthogonalize(x, steps=steps, out_dtype=dt)
    B.check_orth(got, x, steps, MUON, 1e-7, label="plain")
    assert torch.equal(got, ctx.orthogonalize(x, steps=steps, out_dtype=dt)), "two launches differ"
    # an update of weights in place, in a buffer whose rest is left alone
    wide = torch.full((batch, m + 2, n + 7), 7.0, dtype=dt, device="cuda")
    w = wide[:, 1:m + 1, 3:3 + n]
    w.copy_(torch.from_numpy(rng.standard_normal((batch, m, n)) / np.sqrt(n)).to(dt))
    before = w.clone()
    ctx.orthogonalize(x, steps=steps, base=w, out=w, scale=-0.5, keep=0.75)
    B.check_orth(w, x, steps, MUON, 1e-7, before, -0.5, 0.75, "update")
    wide[:, 1:m + 1, 3:3 + n] = 7
    assert (wide == 7).all()


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1.0, 1e25])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_orthogonalize_sizes(ctx, size, dtype):
    """A matrix of any size is as orthogonal, until eps counts."""
    rng = np.random.default_rng(11)
    x = _momentum(rng, 1, 100, 160, H.DT[dtype], size=size)[0]
    B.check_orth(ctx.orthogonalize(x, eps=1e-38), x, 5, MUON, 1e-38)
    B.check_orth(ctx.orthogonalize(x, eps=1e-7), x, 5, MUON, 1e-7)


def test_orthogonalize_is_nearly_orthogonal(ctx):
    """Five steps take the singular values of a random square matrix above 0.01 of its
    norm's into (0.6, 1.3)."""
    rng = np.random.default_rng(12)
    u, _ = np.linalg.qr(rng.standard_normal((200, 200)))
    v, _ = np.linalg.qr(rng.standard_normal((200, 200)))
    x = torch.from_numpy((u * np.linspace(0.2, 1, 200)) @ v).to(torch.bfloat16).cuda()
    s = np.linalg.svd(H.d64(ctx.orthogonalize(x)).numpy(), compute_uv=False)
    assert s.min() > 0.6 and s.max() < 1.3


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_orthogonalize_zero_nan_and_infinity(ctx, dtype):
    rng = np.random.default_rng(13)
    x = _momentum(rng, 4, 70, 90, H.DT[dtype])
    y = ctx.orthogonalize(x)
    z = x.clone()
    z[0] = 0
    z[1, 3, 4] = float("nan")
    z[2, 69, 89] = float("inf")
    got = ctx.orthogonalize(z)
    assert (got[0] == 0).all() and torch.isnan(got[1]).all() and torch.isnan(got[2]).all()
    assert torch.equal(got[3], y[3])


def test_orthogonalize_coefficients_of_each_step(ctx):
    rng = np.random.default_rng(14)
    x = _momentum(rng, 1, 120, 90, torch.float32)[0]
    cs = [(3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (1.875, -1.25, 0.375)]
    B.check_orth(ctx.orthogonalize(x, steps=3, coefficients=cs), x, 3, cs, 1e-7)


def test_orthogonalize_shared_input(ctx):
    """A batch whose inputs are one matrix (a stride of 0)."""
    rng = np.random.default_rng(15)
    x = _momentum(rng, 1, 40, 50, torch.bfloat16)
    got = ctx.orthogonalize(x.expand(3, 40, 50))
    assert torch.equal(got[0], ctx.orthogonalize(x[0])) and torch.equal(got[2], got[0])


# ------------------------------------------------- streams, graphs, refusals
def _calls(ctx, rng):
    x = H.matrix(rng, 70, 256, torch.bfloat16)
    w = H.matrix(rng, 256, 256, torch.bfloat16, 1 / 16)
    n = ctx.prepare_layer_norm(x, want_stats=True)
    qw = ctx.prepare_quantize_rows(w)
    y = ctx.prepare_linear_int8(n.out, qw.q, qw.scale, activation="silu", residual=x)
    nb = ctx.prepare_layer_norm_backward(y.out, x, mean=n.mean, rstd=n.rstd, residual=y.out,
                                         want_bias=True)
    o = ctx.prepare_orthogonalize(w, base=w, scale=-0.1, keep=0.9)
    o2 = ctx.prepare_orthogonalize(w, out_dtype=torch.float32)
    return x, w, [n, qw, y, nb, o, o2]


def _results(calls):
    return [t.clone() for c in calls for t in c.outputs().values()]


def test_another_stream(ctx):
    rng = np.random.default_rng(21)
    x, w, calls = _calls(ctx, rng)
    for c in calls:
        c.launch()
    want = _results(calls)
    for c in calls:
        for t in c.outputs().values():
            t.zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for c in calls:
            c.launch()
        got = _results(calls)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_streams_at_once(ctx):
    """Two programs' calls side by side, each with its own workspace."""
    runs = [_calls(ctx, np.random.default_rng(s)) for s in (31, 32)]
    want = []
    for _, _, calls in runs:
        for c in calls:
            c.launch()
        want.append(_results(calls))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(5):
        for s, (_, _, calls) in zip(streams, runs):
            with torch.cuda.stream(s):
                for c in calls:
                    c.launch()
    torch.cuda.synchronize()
    for w, (_, _, calls) in zip(want, runs):
        assert all(torch.equal(a, b) for a, b in zip(w, _results(calls)))


def test_graph_replays(ctx):
    """A run of all operators captured once and replayed on new inputs, with eager work
    between the replays."""
    rng = np.random.default_rng(22)
    x, w, calls = _calls(ctx, rng)
    for c in calls:
        c.launch()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for c in calls:
            c.launch()
    for i in range(4):
        x.copy_(H.matrix(rng, 70, 256, torch.bfloat16))
        w.copy_(H.matrix(rng, 256, 256, torch.bfloat16, 1 / 16))
        for c in calls:
            c.launch()
        want = _results(calls)
        for c in calls:
            for t in c.outputs().values():
                t.zero_()
        g.replay()
        got = _results(calls)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), f"replay {i}"


def test_offsets_past_32_bits(ctx):
    """Rows more than 2^32 bytes apart from the first."""
    n, stride = 96, 1 << 29
    buf = torch.empty(9 * stride + n, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((10, n), (stride, 1))
    rng = np.random.default_rng(23)
    dense = H.matrix(rng, 10, n, torch.bfloat16)
    x.copy_(dense)
    w, ws = _quantized(rng, 40, n, "dense")
    p, q = ctx.prepare_layer_norm(x, want_stats=True), ctx.prepare_layer_norm(dense, want_stats=True)
    p.launch()
    q.launch()
    assert torch.equal(p.out, q.out)
    a, b = (ctx.prepare_layer_norm_backward(dense, t, mean=p.mean, rstd=p.rstd) for t in (x, dense))
    a.launch()
    b.launch()
    assert torch.equal(a.d_x, b.d_x) and torch.equal(a.d_weight, b.d_weight)
    assert torch.equal(ctx.quantize_rows(x)[0], ctx.quantize_rows(dense)[0])
    assert torch.equal(ctx.linear_int8(x, w, ws), ctx.linear_int8(dense, w, ws))
    assert torch.equal(ctx.orthogonalize(x), ctx.orthogonalize(dense))
    into = buf.as_strided((10, 40), (stride, 1))
    want = ctx.linear_int8(dense, w, ws)
    ctx.linear_int8(dense, w, ws, out=into)
    assert torch.equal(into, want)


def test_refusals(ctx):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    q, s = torch.zeros((8, 64), dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    st = torch.zeros(4, device="cuda")
    for bad in (lambda: ctx.layer_norm(x.t()),
                lambda: ctx.layer_norm(x.double()),
                lambda: ctx.layer_norm(x, weight=torch.ones(64, device="cuda")),
                lambda: ctx.layer_norm(x, bias=torch.ones(63, dtype=x.dtype, device="cuda")),
                lambda: ctx.layer_norm(x.cpu()),
                lambda: ctx.prepare_layer_norm_backward(x[:3], x, mean=st, rstd=st),
                lambda: ctx.prepare_layer_norm_backward(x, x, mean=st[:3], rstd=st),
                lambda: ctx.quantize_rows(x, q=q[:4].float()),
                lambda: ctx.linear_int8(x, x, s),
                lambda: ctx.linear_int8(x, q[:, :63], s),
                lambda: ctx.linear_int8(x, q, s[:7]),
                lambda: ctx.linear_int8(q[:4], q, s),
                lambda: ctx.linear_int8(x, q, s, x_scale=s[:4]),
                lambda: ctx.linear_int8(x, q, s, out_dtype=torch.float16),
                lambda: ctx.orthogonalize(x[0]),
                lambda: ctx.orthogonalize(x, coefficients=[MUON] * 4),
                lambda: ctx.orthogonalize(x, base=x[:3]),
                lambda: ctx.orthogonalize(x[None][:0]),
                lambda: ctx.orthogonalize(x, base=x.float(), out_dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ctx.layer_norm(x, eps=0.0),
                lambda: ctx.prepare_layer_norm_backward(x, x, mean=st, rstd=st, want_x=False,
                                                        want_weight=False).launch(),
                lambda: ctx.orthogonalize(x, steps=0),
                lambda: ctx.orthogonalize(x, steps=65),
                lambda: ctx.orthogonalize(x, eps=0.0),
                lambda: ctx.orthogonalize(x, scale=float("nan")),
                lambda: ctx.orthogonalize(x, coefficients=(3.4445, 4.7750, 2.0315))):
        with pytest.raises(_ffi.LsampError):
            bad()


def test_layer_norm_larger_than_the_caches(ctx):
    """Results of 256 MiB and more, stored past the caches, equal those of their parts."""
    rng = np.random.default_rng(41)
    rows, n = 32800, 4100
    part = H.matrix(rng, 1025, n, torch.bfloat16)
    x = part.repeat(32, 1)
    assert x.shape[0] == rows
    d = x.flip(1).contiguous()
    w, b = (H.matrix(rng, 1, n, torch.bfloat16)[0] for _ in range(2))
    p = ctx.prepare_layer_norm(x, weight=w, bias=b, want_stats=True)
    p.launch()
    q = ctx.prepare_layer_norm_backward(d, x, mean=p.mean, rstd=p.rstd, weight=w, residual=x)
    q.launch()
    few = ctx.prepare_layer_norm(part, weight=w, bias=b, want_stats=True)
    few.launch()
    back = ctx.prepare_layer_norm_backward(d[:1025], part, mean=few.mean, rstd=few.rstd, weight=w,
                                           residual=part)
    back.launch()
    assert torch.equal(p.out.view(32, 1025, n), few.out.expand(32, 1025, n))
    assert torch.equal(q.d_x.view(32, 1025, n), back.d_x.expand(32, 1025, n))
    # 32 equal parts: 32 times their sum, with norm_grads64's roundings of all rows
    D = H.d64(d[:1025])
    terms = D * (H.d64(part) - H.d64(few.mean)[:, None]) * H.d64(few.rstd)[:, None]
    err = (64 + rows // 256 + 64 + 4) * H.E * 32 * terms.abs().sum(0)
    H.check(q.d_weight, B.rounded(32 * terms.sum(0), err, torch.bfloat16), "d_weight")
