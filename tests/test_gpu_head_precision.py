"""What the hidden-state operators' functions and scales may be off by, on the GPU
against 64 bits: rows without a loss beside a float16 gradient's scale."""
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
    rows, ids = torch.arange(m), torch.arange(v)
    want = S.head_grads(d, x, w, t, f.lse, None, 0.0, rows, ids)
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
