"""8-bit products whose rows' scales have a product that is no normal float32 while the results
are: tiny rows by tiny ones, huge by huge, and tiny by huge, through every kind of kernel."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import blocks_common as B
import head_common as H

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lsamp.api import Context
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    c = Context(0, max_rows=4, max_vocab=1024)
    yield c
    c.close()


SHAPES = [
    # rows, in, out: quantised by every work-group; kept in LDS (a block, several, a wave's own
    # columns, lines); too long to be kept; tiles, whole and in parts, of rows that end anywhere
    (2, 300, 70), (9, 300, 70), (4, 1100, 9001), (40, 2000, 33001), (3, 260, 65701),
    (40, 9000, 70), (70, 200, 72), (70, 201, 73), (70, 8208, 72), (2100, 160, 2100),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_results_of_tiny_rows(ctx, shape, dtype):
    """Scales of about 2^-76 each: their product is below 2^-149, a sum times both is not."""
    rows, k, n = shape
    rng = np.random.default_rng(rows + k + n)
    q = torch.from_numpy(rng.integers(64, 128, (rows, k))).to(torch.int8)
    w = torch.from_numpy(rng.integers(64, 128, (n, k))).to(torch.int8)
    x = (q.float() * 2.0 ** -69).to(dtype)
    x[:, 0] = 127 * 2.0 ** -69
    ws = torch.from_numpy(rng.uniform(1, 2, n)).float() * 2.0 ** -74
    ws[0], ws[-1] = 1.0, 2.0 ** 40  # (beside ordinary ones)
    x, w, ws = x.cuda(), w.cuda(), ws.cuda()
    q, xs = B.quantize64(x)
    want = B.int8_64(q, xs, w, ws, dtype=dtype)
    assert float(want[0].min()) > 2.0 ** -126
    assert float((xs.max() * ws[1:-1].max())) < 2.0 ** -126
    H.check(ctx.linear_int8(x, w, ws), want, "out")
    H.check(ctx.linear_int8(q.cuda(), w, ws, x_scale=xs.cuda(), out_dtype=dtype), want, "given")


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_sums_of_zero_of_huge_rows(ctx, shape):
    """Scales whose product is an infinity: a sum of 0 is 0, others infinite."""
    rows, k, n = shape
    w = torch.full((n, k), 100, dtype=torch.int8, device="cuda")
    w[:, 1::2] = -100
    x = torch.full((rows, k), 2.0 ** 100, device="cuda")
    x[:, k // 2 * 2:] = 0  # (as many of either sign)
    x[1, 0] = 2.0 ** 99
    ws = torch.full((n,), 2.0 ** 90, device="cuda")
    got = ctx.linear_int8(x, w, ws)
    assert (got[1] == -float("inf")).all()
    assert (got[0] == 0).all() and (got[2:] == 0).all()
