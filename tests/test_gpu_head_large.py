"""The hidden-state operators on the GPU at sizes of several tiles, pieces and
parts, on sampled rows and columns against 64 bits (head_sampled.py)."""
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


def matrix(rng, rows, cols, dt, std=1.0):
    """Drawn on the GPU: millions of elements."""
    g = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    return (torch.randn((rows, cols), generator=g, device="cuda") * std).to(dt)


def _loss_inputs(rng, dtype, m, k, v):
    dt = H.DT[dtype]
    x, w = matrix(rng, m, k, dt), matrix(rng, v, k, dt, 3 / np.sqrt(k))
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
