"""The hidden-state operators on the GPU against 64-bit restatements
(head_common.py): linear blocks, the vocabulary head's loss, their gradients,
dropout; sizes from 1 to some hundreds, odd ones, any alignment, masked and
ignored rows, infinities and NaN, streams, graphs, and refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import head_common as H
from lsamp import _ffi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lsamp.api import Context
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    c = Context(0, max_rows=4, max_vocab=1024)
    yield c
    c.close()


# --------------------------------------------------------------------- linear
LINEAR = [
    # rows, in, out, activation, bias, residual, layout
    (1, 1, 1, "none", False, False, "dense"),
    (1, 7, 5, "relu", True, True, "odd"),
    (1, 256, 300, "silu", True, True, "dense"),
    (2, 64, 64, "gelu", True, False, "pad"),
    (5, 136, 67, "gelu_tanh", False, True, "dense"),
    (16, 320, 129, "softcap", True, True, "pad"),
    (17, 65, 130, "silu", True, True, "odd"),
    (33, 1000, 96, "none", True, False, "dense"),
    (64, 200, 257, "relu", False, True, "dense"),
    (65, 512, 64, "gelu", True, True, "pad"),
    (100, 33, 1029, "softcap", True, False, "dense"),
    (129, 200, 257, "gelu_tanh", True, True, "odd"),
    (300, 1032, 520, "silu", False, False, "dense"),
    (515, 72, 264, "none", True, True, "dense"),
    (70, 4104, 72, "gelu", True, True, "dense"),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", LINEAR, ids=lambda c: "-".join(map(str, c)))
def test_linear(ctx, case, dtype):
    rows, k, n, act, bias, residual, layout = case
    print(f"linear {case} {dtype}", flush=True)
    rng = np.random.default_rng(rows * 1000003 + k * 1009 + n)
    dt = H.DT[dtype]
    x = H.matrix(rng, rows, k, dt, layout=layout)
    w = H.matrix(rng, n, k, dt, 1 / np.sqrt(k), layout)
    b = H.matrix(rng, 1, n, dt)[0] if bias else None
    res = H.matrix(rng, rows, n, dt, layout=layout) if residual else None
    want = H.linear64(x, w, b, res, act, 5.0)
    p = ctx.prepare_linear(x, w, bias=b, residual=res, activation=act, softcap=5.0, want_pre=True)
    p.launch()
    first = p.out.clone()
    p.launch()
    H.check(p.out, want["out"], "out")
    H.check(p.pre, want["pre"], "pre")
    assert torch.equal(first, p.out), "two launches differ"
    # float32 out, into a padded buffer whose rest is left alone
    wide = torch.full((rows, n + 5), 7.0, device="cuda")
    q = ctx.prepare_linear(x, w, bias=b, residual=res, activation=act, softcap=5.0,
                           out=wide[:, 2:2 + n])
    q.launch()
    H.check(q.out, H.linear64(x, w, b, res, act, 5.0, torch.float32)["out"], "float32 out")
    assert (wide[:, :2] == 7).all() and (wide[:, 2 + n:] == 7).all()


def test_linear_residual_in_place(ctx):
    rng = np.random.default_rng(5)
    x, w = H.matrix(rng, 40, 96, torch.bfloat16), H.matrix(rng, 96, 96, torch.bfloat16, 0.1)
    y = ctx.linear(x, w, activation="silu", residual=x)
    z = x.clone()
    ctx.linear(x, w, activation="silu", residual=z, out=z)
    assert torch.equal(y, z)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_linear_infinities_and_nan(ctx, dtype):
    """A row with a NaN or an infinity changes no other row."""
    rng = np.random.default_rng(6)
    dt = H.DT[dtype]
    x, w = H.matrix(rng, 70, 130, dt), H.matrix(rng, 90, 130, dt)
    clean = ctx.linear(x, w)
    x[3, 129] = float("nan")
    x[66, 0] = float("inf")
    out = ctx.linear(x, w)
    keep = torch.ones(70, dtype=torch.bool)
    keep[[3, 66]] = False
    assert torch.equal(out[keep.cuda()], clean[keep.cuda()])
    assert torch.isnan(out[3]).all()
    want = torch.where(w[:, 0] > 0, float("inf"), float("-inf")).to(dt)
    assert torch.equal(out[66], torch.where(w[:, 0] == 0, torch.full_like(want, float("nan")), want))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", LINEAR, ids=lambda c: "-".join(map(str, c)))
def test_linear_backward(ctx, case, dtype):
    rows, k, n, act, bias, _, layout = case
    print(f"linear backward {case} {dtype}", flush=True)
    rng = np.random.default_rng(rows * 7919 + k * 31 + n)
    dt = H.DT[dtype]
    x = H.matrix(rng, rows, k, dt, layout=layout)
    w = H.matrix(rng, n, k, dt, 1 / np.sqrt(k), layout)
    d = H.matrix(rng, rows, n, dt, layout=layout)
    f = ctx.prepare_linear(x, w, activation=act, softcap=5.0, want_pre=True)
    f.launch()
    p = ctx.prepare_linear_backward(d, x, w, pre=f.pre, activation=act, softcap=5.0,
                                    want_bias=bias)
    p.launch()
    want = H.linear_grads64(d, x, w, f.pre, act, 5.0)
    for name, got in p.outputs().items():
        H.check(got, want[name], name)
    # each gradient alone is the same
    for name in p.outputs():
        kw = {"want_x": name == "d_x", "want_weight": name == "d_weight",
              "want_bias": name == "d_bias"}
        q = ctx.prepare_linear_backward(d, x, w, pre=f.pre, activation=act, softcap=5.0, **kw)
        q.launch()
        assert torch.equal(q.outputs()[name], p.outputs()[name]), name


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "softcap"])
def test_linear_gradient_against_differences(ctx, act):
    """<d, f(x + h v) - f(x - h v)> / 2h against <d_x, v>, <d_weight, v>: float32
    outputs of size ~1 rounded to 2^-24 give differences good to about
    sqrt(rows n) 2^-23 / h, and the third derivative adds h^2."""
    rng = np.random.default_rng(8)
    rows, k, n, h = 24, 40, 56, 2.0 ** -7
    x, w = H.matrix(rng, rows, k, torch.float32), H.matrix(rng, n, k, torch.float32, k ** -0.5)
    d = H.matrix(rng, rows, n, torch.float32)
    f = ctx.prepare_linear(x, w, activation=act, softcap=2.0, want_pre=True)
    f.launch()
    g = ctx.prepare_linear_backward(d, x, w, pre=f.pre, activation=act, softcap=2.0)
    g.launch()
    for name, t in (("d_x", x), ("d_weight", w)):
        v = H.matrix(rng, *t.shape, torch.float32, 1 / np.sqrt(k))
        at = [ctx.linear(*((t + s * h * v, w) if t is x else (x, t + s * h * v)), activation=act,
                         softcap=2.0) for s in (1, -1)]
        diff = float((d.double() * (at[0].double() - at[1].double())).sum() / (2 * h))
        mine = float((g.outputs()[name].double() * v.double()).sum())
        # sums of rows * n terms of size ~1: rounding, then h^2 times third derivatives (< 4)
        tol = np.sqrt(rows * n) * (k * 2.0 ** -22 / h + 4 * h * h)
        assert abs(diff - mine) <= tol, (name, diff, mine, tol)


# ------------------------------------------------------------------ head loss
LOSS = [
    # rows, hidden, vocab, softcap, bias, layout
    (1, 8, 1, 0.0, False, "dense"),
    (1, 64, 257, 0.0, True, "dense"),
    (2, 33, 100, 0.0, False, "odd"),
    (7, 128, 1003, 30.0, True, "pad"),
    (20, 264, 2048, 0.0, False, "dense"),
    (33, 96, 4099, 2.0, True, "dense"),
    (64, 200, 777, 0.0, True, "odd"),
    (65, 136, 1500, 30.0, False, "pad"),
    (130, 320, 640, 0.0, True, "dense"),
    (300, 72, 3001, 30.0, True, "odd"),
]


def _loss_inputs(case, dtype, seed=0):
    rows, k, v, cap, bias, layout = case
    rng = np.random.default_rng(rows * 101 + k * 13 + v + seed)
    dt = H.DT[dtype]
    x = H.matrix(rng, rows, k, dt, layout=layout)
    w = H.matrix(rng, v, k, dt, 3 / np.sqrt(k), layout)
    b = H.matrix(rng, 1, v, dt, 0.5)[0] if bias else None
    t = torch.from_numpy(rng.integers(0, v, rows).astype(np.int32))
    t[rows // 2::5] = -100
    d = torch.from_numpy(rng.uniform(0.5, 2.0, rows).astype(np.float32)) / rows
    return x, w, b, t.cuda(), d.cuda(), cap


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", LOSS, ids=lambda c: "-".join(map(str, c)))
def test_head_loss_and_gradient(ctx, case, dtype):
    print(f"head loss {case} {dtype}", flush=True)
    x, w, b, t, d, cap = _loss_inputs(case, dtype)
    f = ctx.prepare_head_loss(x, w, t, bias=b, softcap=cap)
    f.launch()
    want = H.loss64(x, w, t, b, cap)
    H.check(f.lse, want["lse"], "lse")
    H.check(f.loss, want["loss"], "loss")
    assert not f.row_flags.any()
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, bias=b, softcap=cap, want_bias=True)
    p.launch()
    first = {k: v.clone() for k, v in p.outputs().items()}
    p.launch()
    want = H.loss_grads64(d, x, w, t, f.lse, b, cap)
    for name, got in p.outputs().items():
        H.check(got, want[name], name)
        assert torch.equal(got, first[name]), f"two launches differ in {name}"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_head_loss_in_pieces(ctx, dtype):
    """More columns than a piece of the vocabulary holds, in both directions,
    with rows that have to be laid out first; unequal last pieces."""
    for case in ((5, 501, 70001, 0.0, True, "odd"), (1030, 24, 70000, 0.0, True, "dense")):
        print(f"pieces {case} {dtype}", flush=True)
        x, w, b, t, d, cap = _loss_inputs(case, dtype)
        f = ctx.prepare_head_loss(x, w, t, bias=b, softcap=cap)
        f.launch()
        want = H.loss64(x, w, t, b, cap)
        H.check(f.lse, want["lse"], "lse")
        H.check(f.loss, want["loss"], "loss")
        p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, bias=b, softcap=cap,
                                           want_bias=True)
        p.launch()
        want = H.loss_grads64(d, x, w, t, f.lse, b, cap)
        for name, got in p.outputs().items():
            H.check(got, want[name], name)


@pytest.mark.parametrize("dtype,case", [
    ("bf16", (1030, 8193, 8200, 0.0, True, "odd")), ("f32", (1030, 4101, 8200, 0.0, False, "odd"))])
def test_head_loss_weight_copied_in_pieces(ctx, dtype, case):
    """Weight rows of odd lengths under many rows of x are laid out a piece of
    the vocabulary at a time, in both directions; here two pieces."""
    print(f"copied pieces {case} {dtype}", flush=True)
    x, w, b, t, d, cap = _loss_inputs(case, dtype)
    f = ctx.prepare_head_loss(x, w, t, bias=b, softcap=cap)
    f.launch()
    want = H.loss64(x, w, t, b, cap)
    H.check(f.lse, want["lse"], "lse")
    H.check(f.loss, want["loss"], "loss")
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, bias=b, softcap=cap, want_bias=True)
    p.launch()
    print("the 64-bit gradients", flush=True)
    want = H.loss_grads64(d, x, w, t, f.lse, b, cap)
    for name, got in p.outputs().items():
        H.check(got, want[name], name)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_head_loss_masked_vocabulary(ctx, dtype):
    """Ids with a bias of -inf or the type's lowest value have no mass; whole
    tiles of them; a target among them; every id but one; every id."""
    dt = H.DT[dtype]
    case = (9, 64, 900, 0.0, True, "dense")
    for name in ("some", "lowest", "tiles", "one", "all"):
        print(f"masked {name} {dtype}", flush=True)
        x, w, b, t, d, cap = _loss_inputs(case, dtype)
        keep = t[t >= 0]
        if name == "some":
            b[::3] = float("-inf")
        elif name == "lowest":
            b[100:700] = torch.finfo(dt).min
        elif name == "tiles":
            b[:600] = float("-inf")
        elif name == "one":
            b[:] = float("-inf")
            b[int(keep[0])] = 0
        else:
            b[:] = float("-inf")
        f = ctx.prepare_head_loss(x, w, t, bias=b)
        f.launch()
        p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, bias=b, want_bias=True)
        p.launch()
        if name == "all":
            assert torch.isneginf(f.lse).all()
            assert torch.equal(torch.isnan(f.loss), t >= 0) and (f.loss[t < 0] == 0).all()
            assert (f.row_flags == _ffi.ROW_EMPTY).all()
            for k, g in p.outputs().items():
                assert (g == 0).all(), k
            continue
        assert not f.row_flags.any()
        z, err, _ = H.logits64(x, w, b, 0.0)
        lse = torch.logsumexp(z, 1)
        live = b.cpu().double() > float(torch.finfo(dt).min) / 2
        live_err = err[:, live].amax(1)
        H.check(f.lse, (lse, live_err + 2.0 ** -24 * (256 + 4 * lse.abs())), "lse")
        tt = t.cpu().long()
        zt = z.gather(1, tt.clamp(min=0)[:, None])[:, 0]
        want = torch.where(tt < 0, torch.zeros_like(lse), lse - zt)
        tol = 2 * live_err + 2.0 ** -24 * (512 + 8 * lse.abs() + 4 * zt.abs().nan_to_num(posinf=0, neginf=0))
        H.check(f.loss, (want, tol), "loss")
        if name == "lowest":
            # (the logits of masked ids differ from the lowest value by a rounding of
            # that size: only their absence from the sums is checked)
            assert torch.isfinite(p.d_x.float()).all()
            assert (p.d_bias[100:700][~torch.isin(torch.arange(100, 700), tt).cuda()] == 0).all()
            continue
        grads = H.loss_grads64(d, x, w, t, f.lse, b)
        for k, g in p.outputs().items():
            H.check(g, grads[k], k)


def test_head_loss_flags(ctx):
    """NaN and infinite rows, targets past the vocabulary: flagged, and no other row sees them."""
    case = (70, 64, 300, 0.0, False, "dense")
    x, w, _, t, d, _ = _loss_inputs(case, "bf16")
    t[:] = t.clamp(min=0)
    clean = ctx.head_loss(x, w, t)["loss"].clone()
    t[2], t[3], t[4] = 300, 2 ** 31 - 1, -(2 ** 31)
    x[5, 0] = float("nan")
    x[6, :] = 0
    x[6, 1] = float("inf")
    w[:, 1] = w[:, 1].abs() + 0.1
    f = ctx.prepare_head_loss(x, w, t)
    f.launch()
    flags = f.row_flags.cpu()
    want = torch.zeros(70, dtype=torch.int32)
    want[[2, 3]] = _ffi.ROW_TOKEN_RANGE
    want[[5, 6]] = _ffi.ROW_NONFINITE
    assert torch.equal(flags, want)
    assert torch.isnan(f.loss[[2, 3, 5, 6]]).all() and f.loss[4] == 0
    rest = torch.ones(70, dtype=torch.bool)
    rest[2:7] = False
    assert torch.isfinite(f.loss[rest.cuda()]).all()
    # rows without a loss have no gradient; the others are as if they were alone
    x[5], x[6] = 0, 0
    f.launch()
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse)
    p.launch()
    assert (p.d_x[2:5] == 0).all()
    grads = H.loss_grads64(d, x, w, t, f.lse)
    for k, g in p.outputs().items():
        H.check(g, grads[k], k)
    assert torch.isfinite(clean).all()


def test_head_loss_ignored_rows_only(ctx):
    case = (12, 64, 300, 0.0, False, "dense")
    x, w, _, t, d, _ = _loss_inputs(case, "f16")
    t[:] = -1
    x[3] = float("nan")  # an ignored row's values reach no gradient
    f = ctx.prepare_head_loss(x, w, t)
    f.launch()
    assert (f.loss == 0).all()
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, want_weight=False, want_bias=True)
    p.launch()
    assert (p.d_x == 0).all() and (p.d_bias == 0).all()


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1.0, 1e6])
def test_head_loss_gradient_scales(ctx, scale):
    """A scaled loss gives scaled gradients: small ones are not lost in float16."""
    case = (48, 64, 500, 0.0, False, "dense")
    for dtype in ("f16", "bf16", "f32"):
        x, w, _, t, d, _ = _loss_inputs(case, dtype)
        f = ctx.prepare_head_loss(x, w, t)
        f.launch()
        p = ctx.prepare_head_loss_backward(d * scale, x, w, t, lse=f.lse)
        p.launch()
        if dtype == "f16" and scale == 1e6:
            continue  # (float16 cannot hold the result)
        grads = H.loss_grads64(d * scale, x, w, t, f.lse)
        for k, g in p.outputs().items():
            H.check(g, grads[k], f"{dtype} {k}")


def test_head_loss_gradient_against_differences(ctx):
    """Central differences of the summed loss along random directions, float32:
    the loss rounds to 2^-23 of its size (~8), the third derivative adds h^2."""
    case = (24, 40, 300, 5.0, True, "dense")
    x, w, b, t, d, cap = _loss_inputs(case, "f32")
    f = ctx.prepare_head_loss(x, w, t, bias=b, softcap=cap)
    f.launch()
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, bias=b, softcap=cap, want_bias=True)
    p.launch()
    rng = np.random.default_rng(9)
    h = 2.0 ** -7
    for name, src in (("d_x", x), ("d_weight", w), ("d_bias", b)):
        v = torch.from_numpy((rng.standard_normal(tuple(src.shape)) / np.sqrt(40)).astype(np.float32)).cuda()
        total = []
        for s in (1, -1):
            a = {"d_x": x, "d_weight": w, "d_bias": b}
            a[name] = src + s * h * v
            loss = ctx.head_loss(a["d_x"], a["d_weight"], t, bias=a["d_bias"], softcap=cap)["loss"]
            total.append(float((loss.double() * d.double()).sum()))
        diff = (total[0] - total[1]) / (2 * h)
        mine = float((p.outputs()[name].double() * v.double()).sum())
        tol = float(d.double().sum()) * (40 * 2.0 ** -21 / h + 8 * h * h)
        assert abs(diff - mine) <= tol, (name, diff, mine, tol)


def test_loss_of_logits_and_head_loss_agree(ctx):
    """lsamp_linear's float32 logits through lsamp_logprobs, and lsamp_head_loss."""
    case = (17, 128, 1000, 0.0, True, "dense")
    x, w, b, t, _, _ = _loss_inputs(case, "bf16")
    t[:] = t.clamp(min=0)
    from lsamp.api import Context
    c = Context(0, max_rows=32, max_vocab=1024)
    logits = c.linear(x, w, bias=b, out_dtype=torch.float32)
    chosen = c.logprobs(logits, tokens=t)["chosen"]
    loss = c.head_loss(x, w, t, bias=b)["loss"]
    torch.cuda.synchronize()
    assert float((chosen + loss).abs().max()) <= 2.0 ** -24 * (2 * 128 * 40 + 400)
    c.close()


# -------------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols,p,layout,residual", [
    (1, 1, 0.5, "dense", False), (1, 9, 0.1, "odd", True), (3, 64, 0.25, "dense", True),
    (5, 1001, 0.1, "odd", True), (64, 2048, 0.1, "dense", True), (33, 520, 0.9, "pad", False),
    (7, 4100, 0.05, "pad", True), (300, 24, 0.5, "dense", False), (2, 40, 0.0, "dense", True),
    (2, 40, 1.0, "dense", True), (2, 40, 1.0, "dense", False)])
def test_dropout(ctx, rows, cols, p, layout, residual, dtype):
    rng = np.random.default_rng(rows + cols)
    dt = H.DT[dtype]
    x = H.matrix(rng, rows, cols, dt, layout=layout)
    res = H.matrix(rng, rows, cols, dt, layout=layout) if residual else None
    key, offset = 0x9E3779B97F4A7C15, (3 << 32) + 12345
    out = ctx.dropout(x, p=p, key=key, offset=offset, residual=res)
    keep = H.philox_keep(rows, cols, p, key, offset)
    cut = int(np.rint(np.float64(np.float32(p)) * 65536))
    y = torch.where(keep, H.d64(x) * (65536.0 / max(1, 65536 - cut)), torch.zeros(1, dtype=torch.float64))
    err = 2 * H.E * y.abs()
    if residual:
        y = y + H.d64(res)
        err = err + H.E * y.abs()
    H.check(out, (y, err + H.U[dt] * (y.abs() + err) + H.TINY[dt] * H.U[dt]), "out")
    if not residual:
        assert torch.equal((out != 0).cpu(), keep & (x != 0).cpu())
    # a device step counts as an offset; out may be x
    step = torch.tensor([offset - 7], dtype=torch.int64, device="cuda")
    y2 = x.clone()
    ctx.dropout(y2, p=p, key=key, offset=7, step=step, residual=res, out=y2)
    assert torch.equal(out, y2)


def test_dropout_rate_and_independence(ctx):
    """Kept shares of 2^20 elements within 6 standard deviations, and two offsets
    agree as often as independent masks do."""
    x = torch.ones(512, 2048, dtype=torch.bfloat16, device="cuda")
    n = x.numel()
    masks = [ctx.dropout(x, p=0.3, key=5, offset=o) != 0 for o in (0, 1, 2)]
    masks.append(ctx.dropout(x, p=0.3, key=6, offset=0) != 0)
    q = 1 - round(0.3 * 65536) / 65536
    for m in masks:
        assert abs(float(m.double().mean()) - q) <= 6 * np.sqrt(q * (1 - q) / n)
    same = q * q + (1 - q) ** 2
    for i in range(4):
        for j in range(i):
            s = float((masks[i] == masks[j]).double().mean())
            assert abs(s - same) <= 6 * np.sqrt(same * (1 - same) / n)


def test_dropout_does_not_use_dropped_values(ctx):
    x = torch.full((8, 64), float("nan"), dtype=torch.float32, device="cuda")
    keep = H.philox_keep(8, 64, 0.5, 1, 2).cuda()
    x[keep] = 1.0
    out = ctx.dropout(x, p=0.5, key=1, offset=2)
    assert torch.equal(out, keep.float() * 2)


# ---------------------------------------------- streams, graphs, large offsets
def test_another_stream(ctx):
    rng = np.random.default_rng(12)
    x, w = H.matrix(rng, 40, 128, torch.bfloat16), H.matrix(rng, 300, 128, torch.bfloat16, 0.1)
    t = torch.arange(40, dtype=torch.int32, device="cuda")
    want, wl = ctx.linear(x, w, activation="gelu"), ctx.head_loss(x, w, t)["loss"]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ctx.linear(x, w, activation="gelu")
        gl = ctx.head_loss(x, w, t)["loss"]
    p = ctx.prepare_linear(x, w, activation="gelu")
    p.launch(stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(want, got) and torch.equal(wl, gl) and torch.equal(want, p.out)


def test_graph_of_a_training_step(ctx):
    """Dropout, block, loss and their gradients captured once; replays see new
    inputs and a new dropout step."""
    rng = np.random.default_rng(13)
    dt = torch.bfloat16
    x, w = H.matrix(rng, 72, 104, dt), H.matrix(rng, 104, 104, dt, 0.1)
    head, b = H.matrix(rng, 1200, 104, dt, 0.1), H.matrix(rng, 1, 104, dt)[0]
    t = torch.from_numpy(rng.integers(0, 1200, 72).astype(np.int32)).cuda()
    d = torch.full((72,), 1 / 72, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    drop = ctx.prepare_dropout(x, p=0.25, key=77, step=step)
    block = ctx.prepare_linear(drop.out, w, bias=b, activation="silu", residual=x, want_pre=True)
    loss = ctx.prepare_head_loss(block.out, head, t)
    dh = ctx.prepare_head_loss_backward(d, block.out, head, t, lse=loss.lse)
    db = ctx.prepare_linear_backward(dh.d_x, drop.out, w, pre=block.pre, activation="silu",
                                     want_bias=True)
    dd = ctx.prepare_dropout(db.d_x, p=0.25, key=77, step=step)
    calls = [drop, block, loss, dh, db, dd]

    def outs():
        return [loss.loss, dh.d_x, dh.d_weight, db.d_x, db.d_weight, db.d_bias, dd.out]

    for c in calls:
        c.launch()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for c in calls:
            c.launch()
    for i in range(4):
        x.copy_(H.matrix(rng, 72, 104, dt))
        step.fill_(i)
        for c in calls:
            c.launch()
        torch.cuda.synchronize()
        want = [o.clone() for o in outs()]
        for o in outs():
            o.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, o in zip(want, outs()):
            assert torch.equal(a, o), f"replay {i}"


def test_offsets_past_32_bits(ctx):
    """Matrices whose last rows start past 2^32 bytes and 2^31 elements."""
    dt = torch.bfloat16
    rows, k, n = 40, 64, 48
    ld = (1 << 31) // 32 + 64  # row 32 starts past 2^31 elements
    big = torch.empty(rows * ld, dtype=dt, device="cuda")
    x = big.as_strided((rows, k), (ld, 1))
    rng = np.random.default_rng(14)
    small = H.matrix(rng, rows, k, dt)
    x.copy_(small)
    w = H.matrix(rng, n, k, dt, 0.1)
    assert torch.equal(ctx.linear(x, w), ctx.linear(small, w))
    t = torch.arange(rows, dtype=torch.int32, device="cuda")
    assert torch.equal(ctx.head_loss(x, w, t)["loss"], ctx.head_loss(small, w, t)["loss"])
    out = big.as_strided((rows, n), (ld, 1), 64)
    ctx.linear(small, w, out=out)
    assert torch.equal(out, ctx.linear(small, w))
    assert torch.equal(ctx.dropout(x, p=0.5, key=1), ctx.dropout(small, p=0.5, key=1))


# ------------------------------------------------------------------- refusals
def test_refusals(ctx):
    rng = np.random.default_rng(15)
    x, w = H.matrix(rng, 4, 64, torch.bfloat16), H.matrix(rng, 32, 64, torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    d = H.matrix(rng, 4, 32, torch.bfloat16)
    lse = torch.zeros(4, device="cuda")
    bad = [
        lambda: ctx.linear(x, w[:, :32]),
        lambda: ctx.linear(x, w.float()),
        lambda: ctx.linear(x.double(), w.double()),
        lambda: ctx.linear(x.cpu(), w),
        lambda: ctx.linear(x.t(), w),
        lambda: ctx.linear(x, w, activation="tanh"),
        lambda: ctx.linear(x, w, bias=torch.zeros(31, dtype=torch.bfloat16, device="cuda")),
        lambda: ctx.linear(x, w, residual=x),
        lambda: ctx.linear(x, w, out_dtype=torch.float16),
        lambda: ctx.head_loss(x, w, t.long()),
        lambda: ctx.head_loss(x, w, t[:3]),
        lambda: ctx.prepare_linear_backward(d, x, w, pre=d, activation="silu"),
        lambda: ctx.prepare_head_loss_backward(lse, x, w, t, lse=lse[:3]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print(f"call {i} was taken")
    refused = [
        (lambda: ctx.linear(x, w, activation="softcap", softcap=0.0), _ffi.LSAMP_ERR_INVALID_ARGUMENT),
        (lambda: ctx.linear(x, w, activation="softcap", softcap=float("nan")), _ffi.LSAMP_ERR_INVALID_ARGUMENT),
        (lambda: ctx.linear(x[:0], w), _ffi.LSAMP_ERR_SHAPE),
        (lambda: ctx.head_loss(x, w, t, softcap=-1.0), _ffi.LSAMP_ERR_INVALID_ARGUMENT),
        (lambda: ctx.prepare_linear_backward(d, x, w, activation="silu"), _ffi.LSAMP_ERR_INVALID_ARGUMENT),
        (lambda: ctx.prepare_linear_backward(d, x, w, want_x=False, want_weight=False), _ffi.LSAMP_ERR_INVALID_ARGUMENT),
        (lambda: ctx.dropout(x, p=1.5, key=0), _ffi.LSAMP_ERR_INVALID_ARGUMENT),
        (lambda: ctx.dropout(x, p=float("nan"), key=0), _ffi.LSAMP_ERR_INVALID_ARGUMENT),
    ]
    for i, (f, status) in enumerate(refused):
        with pytest.raises(_ffi.LsampError) as e:
            f()
            print(f"call {i} was taken")
        assert e.value.status == status, (i, str(e.value))
    # a workspace that is missing or too small is refused before anything runs
    p = ctx.prepare_head_loss(x, w, t)
    p.args.workspace_bytes -= 1
    with pytest.raises(_ffi.LsampError) as e:
        p.launch()
    assert e.value.status == _ffi.LSAMP_ERR_CAPACITY
    p.args.workspace_bytes += 1
    p.launch()
    torch.cuda.synchronize()
