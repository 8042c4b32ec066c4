"""The hidden-state operators on the GPU in every tile shape, with several tiles,
pieces and parts, against 64 bits (head_sampled.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import head_common as H
import head_sampled as S
import head_shapes as SH

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lsamp.api import Context
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    c = Context(0, max_rows=4, max_vocab=1024)
    yield c
    c.close()


def matrix(rng, rows, cols, dt, std=1.0, layout="dense"):
    """Drawn on the GPU (millions of elements), in the layouts of head_common.matrix."""
    g = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    a = (torch.randn((rows, cols), generator=g, device="cuda") * std).to(dt)
    if layout == "dense":
        return a
    extra, shift = (8, 0) if layout == "pad" else (3, 1)
    wide = torch.full((rows, cols + extra), float("nan"), dtype=dt, device="cuda")
    wide[:, shift:shift + cols] = a
    return wide[:, shift:shift + cols]


def _loss_inputs(rng, dtype, m, k, v, layout="dense"):
    dt = H.DT[dtype]
    x, w = matrix(rng, m, k, dt, layout=layout), matrix(rng, v, k, dt, 3 / np.sqrt(k), layout)
    b = matrix(rng, 1, v, dt, 0.5)[0]
    t = torch.from_numpy(rng.integers(0, v, m).astype(np.int32))
    t[m // 2::5] = -100
    d = torch.from_numpy(rng.uniform(0.5, 2.0, m).astype(np.float32)) / m
    return x, w, b, t.cuda(), d.cuda()


@pytest.mark.parametrize("case", [("f32", 614, 512, 129280), ("bf16", 411, 240, 205007),
                                  ("f16", 686, 472, 110778)], ids=lambda c: "-".join(map(str, c)))
def test_parts_of_later_pieces(ctx, case):
    """d_x whose pieces of the vocabulary are split into parts, the last piece
    shorter than the first: every id's share arrives.  A third of the targets are
    among the last 400 ids, the last part's, whose share is most of a row of d_x."""
    print(f"parts of pieces {case}", flush=True)
    dtype, m, k, v = case
    rng = np.random.default_rng(m + v)
    x, w, b, t, d = _loss_inputs(rng, dtype, m, k, v)
    t[::3] = torch.from_numpy(rng.integers(v - 400, v, len(t[::3])).astype(np.int32)).cuda()
    f = ctx.prepare_head_loss(x, w, t, bias=b)
    f.launch()
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, bias=b, want_bias=True)
    p.launch()
    rows, ids = S.sample(rng, m, 40), S.sample(rng, v, 200)
    want = S.head_grads(d, x, w, t, f.lse, b, 0.0, rows, ids)
    H.check(p.d_x[rows.cuda()], want["d_x"], "d_x")
    H.check(p.d_weight[ids.cuda()], want["d_weight"], "d_weight")
    H.check(p.d_bias[ids.cuda()], want["d_bias"], "d_bias")


def test_gradients_of_rows_past_8_mib(ctx):
    """float32 rows of more than 8 MiB: the gradient at the pre-activations is as long."""
    rng = np.random.default_rng(41)
    m, k, n = 130, 64, (1 << 21) + 1
    x, w = matrix(rng, m, k, torch.float32), matrix(rng, n, k, torch.float32, 1 / 8)
    d, pre = matrix(rng, m, n, torch.float32), matrix(rng, m, n, torch.float32)
    p = ctx.prepare_linear_backward(d, x, w, pre=pre, activation="silu", want_bias=True)
    p.launch()
    rows, outs = S.sample(rng, m, 3), S.sample(rng, n, 200)
    want = S.linear_grads(d, x, w, pre, "silu", 0.0, rows, outs)
    H.check(p.d_x[rows.cuda()], want["d_x"], "d_x")
    H.check(p.d_weight[outs.cuda()], want["d_weight"], "d_weight")
    H.check(p.d_bias[outs.cuda()], want["d_bias"], "d_bias")


def _typed(cases):
    """Cases of "16" in both 16-bit types."""
    for c in cases:
        for dtype in ("bf16", "f16") if "16" in c else ("f32",):
            yield tuple(dtype if v == "16" else v for v in c)


def _id(c):
    return "-".join(map(str, c))


ACTS = ["none", "silu", "relu", "gelu", "gelu_tanh", "softcap"]


def _linear(ctx, dtype, m, k, n, layout, act, streamed=False):
    rng = np.random.default_rng(m + 3 * k + 7 * n)
    dt = H.DT[dtype]
    x, w = matrix(rng, m, k, dt, layout=layout), matrix(rng, n, k, dt, 1 / np.sqrt(k), layout)
    b, res = matrix(rng, 1, n, dt)[0], matrix(rng, m, n, dt, layout=layout)
    kw = dict(bias=b, activation=act, softcap=5.0)
    p = ctx.prepare_linear(x, w, residual=res, want_pre=streamed, **kw)
    p.launch()
    want = S.linear(x, w, b, res, act, 5.0, dt)
    H.check(p.out, want["out"], "out")
    if streamed:
        H.check(p.pre, want["pre"], "pre")
    # into the residual's own memory; and in float32, into padded rows
    inplace = ctx.prepare_linear(x, w, residual=res, out=res, **kw)
    wide = torch.full((m, n + 5), 7.0, device="cuda")
    bare = ctx.prepare_linear(x, w, out=wide[:, 2:2 + n], **kw)
    bare.launch()
    inplace.launch()
    assert torch.equal(res, p.out), "in place"
    H.check(bare.out, S.linear(x, w, b, None, act, 5.0, torch.float32)["out"], "float32 out")
    assert (wide[:, :2] == 7).all() and (wide[:, 2 + n:] == 7).all()


@pytest.mark.parametrize("case", _typed(c[1:] for c in SH.SHAPES if c[0] == "linear"), ids=_id)
def test_linear_in_every_shape(ctx, case):
    print(f"linear {case}", flush=True)
    _linear(ctx, *case, ACTS[sum(case[1:4]) % 6])


@pytest.mark.parametrize("case", SH.STREAMED, ids=_id)
def test_linear_stored_past_the_caches(ctx, case):
    print(f"streamed {case}", flush=True)
    _linear(ctx, *case, "dense", "silu", streamed=True)


@pytest.mark.parametrize("case", _typed(c[1:] for c in SH.SHAPES if c[0] == "linear_backward"), ids=_id)
def test_linear_gradients_in_every_shape(ctx, case):
    print(f"linear backward {case}", flush=True)
    dtype, m, k, n, layout = case
    rng = np.random.default_rng(m + 3 * k + 7 * n)
    dt = H.DT[dtype]
    act = ACTS[1 + sum(case[1:4]) % 5]
    x, w = matrix(rng, m, k, dt, layout=layout), matrix(rng, n, k, dt, 1 / np.sqrt(k), layout)
    d, pre = matrix(rng, m, n, dt, layout=layout), matrix(rng, m, n, torch.float32)
    p = ctx.prepare_linear_backward(d, x, w, pre=pre, activation=act, softcap=5.0, want_bias=True)
    p.launch()
    want = S.linear_grads(d, x, w, pre, act, 5.0)
    for name, got in p.outputs().items():
        H.check(got, want[name], name)


def _head(ctx, dtype, m, k, v, layout, cap=0.0, sampled=False):
    rng = np.random.default_rng(m + 3 * k + 7 * v)
    x, w, b, t, d = _loss_inputs(rng, dtype, m, k, v, layout)
    if sampled:  # (a third of the targets in the last, short piece)
        t[::3] = v - 1
    f = ctx.prepare_head_loss(x, w, t, bias=b, softcap=cap)
    f.launch()
    p = ctx.prepare_head_loss_backward(d, x, w, t, lse=f.lse, bias=b, softcap=cap, want_bias=True)
    p.launch()
    rows, ids = (S.sample(rng, n, 100) for n in (m, v)) if sampled else (None, None)
    at = slice(None) if rows is None else rows.cuda()
    want = S.loss(x[at], w, t[at], b, cap)
    H.check(f.lse[at], want["lse"], "lse")
    H.check(f.loss[at], want["loss"], "loss")
    assert not f.row_flags.any()
    want = S.head_grads(d, x, w, t, f.lse, b, cap, rows, ids)
    H.check(p.d_x[at], want["d_x"], "d_x")
    at = slice(None) if ids is None else ids.cuda()
    H.check(p.d_weight[at], want["d_weight"], "d_weight")
    H.check(p.d_bias[at], want["d_bias"], "d_bias")


@pytest.mark.parametrize("case", _typed(c[1:] for c in SH.SHAPES if c[0] == "head"), ids=_id)
def test_head_in_every_shape(ctx, case):
    print(f"head {case}", flush=True)
    _head(ctx, *case, cap=(0.0, 20.0)[sum(case[1:4]) % 2])


@pytest.mark.parametrize("case", SH.LAST_PIECES, ids=_id)
def test_head_whose_last_piece_is_short(ctx, case):
    print(f"short last piece {case}", flush=True)
    _head(ctx, "bf16", *case, "dense", sampled=True)


@pytest.mark.parametrize("case", _typed(SH.COPIED), ids=_id)
def test_head_whose_weight_is_copied_in_pieces(ctx, case):
    print(f"copied pieces {case}", flush=True)
    _head(ctx, *case, sampled=True)


def _nonfinite(t, rng):
    """A NaN in one row and an infinity in another, in the last and first columns."""
    a, b = (int(i) for i in rng.choice(t.shape[0], 2, replace=False))
    t[a, -1] = float("nan")
    t[b, 0] = float("inf")
    keep = torch.ones(t.shape[0], dtype=torch.bool)
    keep[[a, b]] = False
    return a, b, keep.cuda()


@pytest.mark.parametrize("case", _typed(c[1:] for c in SH.SHAPES if c[0] == "linear"), ids=_id)
def test_nonfinite_rows_stay_alone_in_every_shape(ctx, case):
    print(f"nonfinite {case}", flush=True)
    dtype, m, k, n, layout = case
    rng = np.random.default_rng(m + k + n)
    dt = H.DT[dtype]
    x, w = matrix(rng, m, k, dt, layout=layout), matrix(rng, n, k, dt, 1 / np.sqrt(k), layout)
    clean = ctx.linear(x, w)
    a, b, keep = _nonfinite(x, rng)
    out = ctx.linear(x, w)
    assert torch.equal(out[keep], clean[keep])
    assert torch.isnan(out[a]).all()
    # (infinity times a weight of 0 is no number)
    assert torch.equal(torch.isnan(out[b]), w[:, 0] == 0)
    assert torch.equal(out[b] > 0, w[:, 0] > 0) and torch.isinf(out[b][w[:, 0] != 0]).all()


@pytest.mark.parametrize("case", _typed(c[1:] for c in SH.SHAPES if c[0] == "linear_backward"), ids=_id)
def test_nonfinite_rows_stay_alone_in_d_x(ctx, case):
    print(f"nonfinite d_out {case}", flush=True)
    dtype, m, k, n, layout = case
    rng = np.random.default_rng(m + k + n)
    dt = H.DT[dtype]
    x, w = matrix(rng, m, k, dt, layout=layout), matrix(rng, n, k, dt, 1 / np.sqrt(k), layout)
    d, pre = matrix(rng, m, n, dt, layout=layout), matrix(rng, m, n, torch.float32).abs() + 0.1
    p = ctx.prepare_linear_backward(d, x, w, pre=pre, activation="relu", want_weight=False)
    p.launch()
    clean = p.d_x.clone()
    a, b, keep = _nonfinite(d, rng)
    p.launch()
    assert torch.equal(p.d_x[keep], clean[keep])
    assert torch.isnan(p.d_x[a]).all()
    assert torch.equal(torch.isnan(p.d_x[b]), w[0] == 0)
    assert torch.equal(p.d_x[b] > 0, w[0] > 0)
