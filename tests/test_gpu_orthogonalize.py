"""Orthogonalised updates on the GPU: bfloat16 results as exact as float32 ones unless the
caller asks for fast products, and what either is off by for matrices of low rank and in many
steps."""
from __future__ import annotations

import pytest
import torch

import orth_common as O
from lsamp import _ffi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lsamp.api import Context
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    c = Context(0, max_rows=4, max_vocab=1024)
    yield c
    c.close()


@pytest.mark.parametrize("shape", [(1, 64, 64), (2, 130, 300), (4, 256, 256), (2, 515, 157)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_bfloat16_results_are_float32_ones_rounded_once(ctx, shape, dtype):
    x = O.momenta(*shape, dtype, seed=sum(shape))
    wide = ctx.orthogonalize(x, out_dtype=torch.float32)
    O.check(wide, x, 5, False, label="float32")
    assert torch.equal(ctx.orthogonalize(x, out_dtype=torch.bfloat16), wide.bfloat16())
    w = torch.randn(shape, device="cuda").bfloat16()
    update = dict(scale=-0.5, keep=0.75)
    wide = ctx.orthogonalize(x, base=w.float(), **update)
    assert torch.equal(ctx.orthogonalize(x, base=w, **update), wide.bfloat16())
    ctx.orthogonalize(x, base=w, out=w, **update)
    assert torch.equal(w, wide.bfloat16())


@pytest.mark.parametrize("shape", [(1, 64, 64), (2, 130, 300), (4, 256, 256), (2, 515, 157)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_fast_products(ctx, shape, dtype):
    x = O.momenta(*shape, dtype, seed=sum(shape) + 1)
    got = ctx.orthogonalize(x, out_dtype=torch.bfloat16, fast=True)
    O.check(got, x, 5, True)
    assert torch.equal(got, ctx.orthogonalize(x, out_dtype=torch.bfloat16, fast=True))
    w = torch.randn(shape, device="cuda").bfloat16()
    before = w.clone()
    ctx.orthogonalize(x, base=w, out=w, scale=-0.5, keep=0.75, fast=True)
    O.check(w, x, 5, True, base=before, scale=-0.5, keep=0.75, label="update")


def _low_rank(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    l, r = (torch.randn(s, generator=g, device="cuda") for s in ((256, 8), (8, 256)))
    return (l @ r)[None].to(dtype)


def _steep(dtype):
    """Singular values from 1 to 1e-6, evenly by their logarithms."""
    g = torch.Generator(device="cuda").manual_seed(4)
    u, v = (torch.linalg.qr(torch.randn((512, 512), generator=g, device="cuda").double())[0]
            for _ in range(2))
    s = torch.logspace(0, -6, 512, dtype=torch.float64, device="cuda")
    return ((u * s) @ v)[None].to(dtype)


@pytest.mark.parametrize("fast", [False, True], ids=["full", "fast"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("matrix,steps", [(_low_rank, 5), (_steep, 5), (_steep, 10)],
                         ids=["rank 8", "steep", "steep, 10 steps"])
def test_singular_matrices_and_many_steps(ctx, matrix, steps, dtype, fast):
    """Directions whose singular values are near 0 leave every step as much larger as its
    slope there, and so does what is off in them."""
    x = matrix(dtype)
    got = ctx.orthogonalize(x, steps=steps, fast=fast,
                            out_dtype=torch.bfloat16 if fast else torch.float32)
    worst = O.check(got, x, steps, fast)
    print(f"{matrix.__name__} {dtype} {steps} steps, fast {fast}: {worst:.2e}", flush=True)


def test_fast_is_refused_for_other_results(ctx):
    x = torch.zeros((64, 64), device="cuda")
    for dt in (torch.float32, torch.float16):
        with pytest.raises(_ffi.LsampError):
            ctx.orthogonalize(x, out_dtype=dt, fast=True)
