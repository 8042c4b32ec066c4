"""A norm's gradients written over x, over d_out and over the residual on the GPU: the same bits
as into another matrix."""
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


@pytest.mark.parametrize("over", ["x", "d_out", "residual"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,n", [(1, 8), (50, 777), (700, 4000), (768, 513), (1200, 300),
                                    (20, 9000), (40, 17000)])
def test_gradients_over(ctx, rows, n, dtype, over):
    rng = np.random.default_rng(rows + n)
    x, d, r = (H.matrix(rng, rows, n, H.DT[dtype]) for _ in range(3))
    w = H.matrix(rng, 1, n, H.DT[dtype])[0]
    p = ctx.prepare_layer_norm(x, weight=w, want_stats=True)
    p.launch()
    kw = dict(mean=p.mean, rstd=p.rstd, weight=w, want_bias=True)
    apart = ctx.prepare_layer_norm_backward(d, x, residual=r, **kw)
    apart.launch()
    want = B.norm_grads64(d, x, p.mean, p.rstd, w, r)
    into = {"x": x, "d_out": d, "residual": r}
    t = {k: v.clone() for k, v in into.items()}
    q = ctx.prepare_layer_norm_backward(t["d_out"], t["x"], residual=t["residual"], d_x=t[over], **kw)
    q.launch()
    assert torch.equal(t[over], apart.d_x)
    assert all(torch.equal(t[k], v) for k, v in into.items() if k != over)
    for name in ("d_weight", "d_bias"):
        H.check(getattr(q, name), want[name], name)
