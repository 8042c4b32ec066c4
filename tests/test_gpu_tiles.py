"""Every tile of the batched products of orthogonalised updates and of the 8-bit products
against 64 bits on the GPU."""
from __future__ import annotations

import pytest
import torch

import head_common as H
import orth_common as O
import tile_shapes as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lsamp.api import Context
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    c = Context(0, max_rows=4, max_vocab=1024)
    yield c
    c.close()


@pytest.mark.parametrize("turned", [False, True], ids=["as it is", "transposed"])
@pytest.mark.parametrize("shape", S.ORTH, ids=lambda s: "x".join(map(str, s)))
def test_orthogonalize(ctx, shape, turned):
    batch, m, n = shape
    if turned:
        m, n = n, m
    print(f"orth {batch} x {m} x {n}", flush=True)
    x = O.momenta(batch, m, n, torch.float32, seed=m + n)
    wide = ctx.orthogonalize(x, steps=2)
    O.check(wide, x, 2, False, label="two parts")
    assert torch.equal(ctx.orthogonalize(x, steps=2, out_dtype=torch.bfloat16), wide.bfloat16())
    assert torch.equal(ctx.orthogonalize(x, steps=2), wide), "two launches differ"
    # an update in place, in a buffer whose rest is left alone
    full = torch.full((batch, m + 2, n + 7), 7.0, dtype=torch.bfloat16, device="cuda")
    w = full[:, 1:m + 1, 3:3 + n]
    g = torch.Generator(device="cuda").manual_seed(n)
    w.copy_(torch.randn((batch, m, n), generator=g, device="cuda") / n ** 0.5)
    before = w.clone()
    ctx.orthogonalize(x, steps=2, base=w, out=w, scale=-0.5, keep=0.75, fast=True)
    O.check(w, x, 2, True, base=before, scale=-0.5, keep=0.75, label="fast")
    full[:, 1:m + 1, 3:3 + n] = 7
    assert (full == 7).all()


def _view(t, layout):
    if layout == "dense":
        return t
    wide = torch.full((t.shape[0], t.shape[1] + 3), 55, dtype=t.dtype, device="cuda")
    wide[:, 1:1 + t.shape[1]] = t
    return wide[:, 1:1 + t.shape[1]]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", S.INT8, ids=lambda c: "-".join(map(str, c)))
def test_linear_int8(ctx, case, dtype):
    rows, k, n, layout = case
    print(f"int8 {case} {dtype}", flush=True)
    dt = H.DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows + k + n)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)
    x = _view(randn(rows, k), layout)
    w = _view(torch.randint(-127, 128, (n, k), generator=g, device="cuda").to(torch.int8), layout)
    ws = torch.rand(n, generator=g, device="cuda").add_(0.5).div_(127 * k ** 0.5)
    b, res = randn(n), _view(randn(rows, n), layout)
    q, xs = ctx.quantize_rows(x)
    # (as int8_64: three roundings of the product, one of each sum, the result's)
    z = (q.double() @ w.double().t().contiguous()) * xs.double()[:, None] * ws.double()
    err = 3 * H.E * z.abs()
    z = z + b.double()
    err = err + H.E * (z.abs() + err)
    y = z.clamp(min=0) + res.double()
    err = 1.2 * err + 16 * H.E * (z.abs() + 1)
    err = err + H.E * (y.abs() + err)

    def check(got, to):
        bound = err + H.U[to] * (y.abs() + err) + H.TINY[to] * H.U[to]
        bad = ~((got.double() - y).abs() <= bound)
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside the bound"
    kw = dict(bias=b, residual=res, activation="relu")
    full = torch.full((rows, n + 5), 7.0, dtype=dt, device="cuda")
    first = full[:, 2:2 + n]
    ctx.linear_int8(x, w, ws, out=first, **kw)
    check(first, dt)
    assert (full[:, :2] == 7).all() and (full[:, 2 + n:] == 7).all()
    assert torch.equal(ctx.linear_int8(x, w, ws, **kw), first), "two launches differ"
    # quantised by the caller, from rows of any alignment: the same bits
    assert torch.equal(ctx.linear_int8(_view(q, layout), w, ws, x_scale=xs, **kw), first)
    check(ctx.linear_int8(x, w, ws, out_dtype=torch.float32, **kw), torch.float32)
