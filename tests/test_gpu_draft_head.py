"""The draft head (lsamp/draft_head.py): its gradients against autograd of the
same network in 64 bits, training that learns, and drafts that are the argmax of
its logits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import head_common as H
from lsamp import workloads as W

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lsamp.api import Context
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    c = Context(0, max_rows=64, max_vocab=2048)
    yield c
    c.close()


def _batch(t, seed=3, tokens=40):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t.targets.copy_(torch.randint(0, tokens, (t.rows,), generator=g, device="cuda").int())
    code = torch.randn((tokens, t.x.shape[1]), generator=g, device="cuda")
    t.x.copy_(code[t.targets.long()] + 0.3 * torch.randn(t.x.shape, generator=g, device="cuda"))


@pytest.mark.parametrize("dropout", [0.0, 0.25])
def test_gradients_are_autograds(ctx, dropout):
    """float32, two blocks: every gradient against autograd of the formulas in 64
    bits, with the same kept elements.  The chain of five products of at most 1,500
    terms rounds to about sqrt(1500) 2^-23 of a gradient's norm a product."""
    from lsamp.draft_head import DraftHead
    m = DraftHead(ctx, 96, 1500, blocks=2, dtype=torch.float32, dropout=dropout, seed=9)
    t = m.training(70)
    _batch(t)
    t.targets[5] = -1
    t.launch()
    step = int(t.step)
    ws = [H.d64(w).requires_grad_() for w in m.weights]
    bs = [H.d64(b).requires_grad_() for b in m.biases]
    head = H.d64(m.head).requires_grad_()
    x = H.d64(t.x)
    for i, (w, b) in enumerate(zip(ws, bs)):
        keep = H.philox_keep(70, 96, dropout, 9, (i << 48) + step)
        scale = 65536.0 / (65536 - round(dropout * 65536))
        x = x + torch.nn.functional.silu((x * keep * scale) @ w.t() + b)
    z = x @ head.t()
    tt = t.targets.cpu().long()
    loss = torch.logsumexp(z, 1) - z.gather(1, tt.clamp(min=0)[:, None])[:, 0]
    loss = torch.where(tt >= 0, loss, torch.zeros_like(loss))
    (loss * H.d64(t.d_loss)).sum().backward()
    want = {"head": head.grad, **{f"weight{i}": w.grad for i, w in enumerate(ws)},
            **{f"bias{i}": b.grad for i, b in enumerate(bs)}}
    tol = 5 * np.sqrt(1500) * 2.0 ** -23
    assert float((H.d64(t.loss) - loss.detach()).abs().max()) <= 64 * 2.0 ** -23 * float(z.detach().abs().max())
    for name, y in want.items():
        off = float((H.d64(t.grads[name]) - y).norm() / y.norm())
        assert off <= tol, (name, off, tol)


def test_training_learns_and_drafts_follow(ctx):
    """A code that names its target is learnt: the loss falls below half of a
    guess among the 40 tokens (log 40), and greedy drafts are the argmax of the logits."""
    from lsamp.draft_head import DraftHead
    m = DraftHead(ctx, 128, 2048, blocks=2, dropout=0.1, seed=4)
    t = m.training(256)
    for step in range(60):
        _batch(t)
        t.launch()
        t.update(2.0)
    assert not t.row_flags.any()
    _batch(t)
    score = m.score(t.x, t.targets)
    assert float(score["loss"].mean()) < 0.5 * np.log(40)
    params = W._params([W.resolve_cbv2(temperature=0.0, vocab=2048)] * 32)
    logits = m.logits(t.x[:32])
    drafts = m.propose(t.x[:32], params, uniforms=torch.zeros(32, device="cuda"))
    assert torch.equal(drafts.long(), logits.float().argmax(1))
