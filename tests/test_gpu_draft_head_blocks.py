"""The draft head with layer norms, orthogonalised updates and 8-bit serving
(lsamp/draft_head.py): gradients against autograd of the same network in 64 bits,
updates against the formula, and 8-bit logits within what quantising may do."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import blocks_common as B
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
    """float32, two blocks with norms: every gradient against autograd of the formulas in
    64 bits, with the same kept elements.  As without norms, the chain of products of at
    most 1,500 terms rounds to about sqrt(1500) 2^-23 of a gradient's norm a product; each
    of three norms' gradients, of at most 96 terms a sum, adds less than a product."""
    from lsamp.draft_head import DraftHead
    m = DraftHead(ctx, 96, 1500, blocks=2, dtype=torch.float32, dropout=dropout, norm=True, seed=9)
    for w, b in m.norms:
        w.add_(0.2 * torch.randn_like(w))
        b.add_(0.1 * torch.randn_like(b))
    t = m.training(70)
    _batch(t)
    t.targets[5] = -1
    t.launch()
    step = int(t.step)
    ws = [H.d64(w).requires_grad_() for w in m.weights]
    bs = [H.d64(b).requires_grad_() for b in m.biases]
    nw = [H.d64(w).requires_grad_() for w, _ in m.norms]
    nb = [H.d64(b).requires_grad_() for _, b in m.norms]
    head = H.d64(m.head).requires_grad_()
    x = H.d64(t.x)

    def norm(i, v):
        return torch.nn.functional.layer_norm(v, (96,), nw[i], nb[i], float(np.float32(1e-5)))
    for i, (w, b) in enumerate(zip(ws, bs)):
        keep = H.philox_keep(70, 96, dropout, 9, (i << 48) + step)
        scale = 65536.0 / (65536 - round(dropout * 65536))
        x = x + torch.nn.functional.silu((norm(i, x) * keep * scale) @ w.t() + b)
    z = norm(2, x) @ head.t()
    tt = t.targets.cpu().long()
    loss = torch.logsumexp(z, 1) - z.gather(1, tt.clamp(min=0)[:, None])[:, 0]
    loss = torch.where(tt >= 0, loss, torch.zeros_like(loss))
    (loss * H.d64(t.d_loss)).sum().backward()
    want = {"head": head.grad}
    for name, ts in (("weight", ws), ("bias", bs), ("norm_weight", nw), ("norm_bias", nb)):
        want.update({f"{name}{i}": v.grad for i, v in enumerate(ts)})
    assert set(want) == set(t.grads)
    tol = 8 * np.sqrt(1500) * 2.0 ** -23
    for name, y in want.items():
        off = float((H.d64(t.grads[name]) - y).norm() / y.norm())
        assert off <= tol, (name, off, tol)


def test_served_and_trained_forward_agree(ctx):
    from lsamp.draft_head import DraftHead
    m = DraftHead(ctx, 128, 1000, blocks=2, norm=True, seed=2)
    t = m.training(40)
    _batch(t)
    t.launch()
    assert torch.equal(m.score(t.x, t.targets)["loss"], t.loss)


def test_orthogonal_update(ctx):
    """Two steps of the blocks' matrices against the formula: each adds orth of the
    gradient with momentum, in float32, to the weights."""
    from lsamp.draft_head import DraftHead
    m = DraftHead(ctx, 96, 500, blocks=2, dtype=torch.float32, norm=True, seed=5)
    t = m.training(200)
    momenta = [torch.zeros(96, 96, dtype=torch.float64) for _ in m.weights]
    for step in range(2):
        _batch(t, seed=step)
        t.launch()
        before = [w.clone() for w in m.weights]
        head = m.head.clone()
        t.update_orthogonal(0.05, plain_rate=0.5, momentum=0.9, decay=0.1)
        for i, w in enumerate(m.weights):
            grad = H.d64(t.grads[f"weight{i}"])
            momenta[i] = 0.9 * momenta[i] + grad
            # (the sum is rounded to float32, as the call's input is)
            x = (grad + 0.9 * momenta[i]).float()
            far = H.d64(t.nesterov[i]) - x.double()
            assert float(far.norm()) <= 4 * H.E * float(x.norm())
            B.check_orth(w, t.nesterov[i], 5, (3.4445, -4.7750, 2.0315), 1e-7, before[i],
                         -float(np.float32(0.05)), float(np.float32(1 - 0.05 * 0.1)))
        assert torch.equal(m.head, head.add(t.grads["head"], alpha=-0.5))


@pytest.mark.parametrize("norm", [False, True])
def test_quantized_head_serves(ctx, norm):
    """The 8-bit head's calls are the operators on its quantised weights, and its drafts
    the argmax of its logits."""
    from lsamp.draft_head import DraftHead
    m = DraftHead(ctx, 128, 2048, blocks=2, norm=norm, seed=4)
    q = m.quantized()
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((32, 128), generator=g, device="cuda").to(m.dtype)
    h = x
    for i, (w, b) in enumerate(zip(m.weights, m.biases)):
        n = ctx.layer_norm(h, weight=m.norms[i][0], bias=m.norms[i][1]) if norm else h
        qw, s = B.quantize64(w)
        qx, xs = B.quantize64(n)
        out = ctx.linear_int8(n, qw.cuda(), s.cuda(), bias=b, activation="silu", residual=h)
        H.check(out, B.int8_64(qx, xs, qw, s, b, h, "silu", 0.0, m.dtype), f"block {i}")
        h = out
    h = ctx.layer_norm(h, weight=m.norms[2][0], bias=m.norms[2][1]) if norm else h
    assert torch.equal(q.forward(x), h)
    logits = q.logits(x)
    qw, s = B.quantize64(m.head)
    qx, xs = B.quantize64(h)
    H.check(logits, B.int8_64(qx, xs, qw, s, dtype=m.dtype), "logits")
    params = W._params([W.resolve_cbv2(temperature=0.0, vocab=2048)] * 32)
    drafts = q.propose(x, params, uniforms=torch.zeros(32, device="cuda"))
    assert torch.equal(drafts.long(), logits.float().argmax(1))
    for call in (lambda: q.training(4), lambda: q.score(x, None)):
        with pytest.raises(TypeError):
            call()


def test_example_runs(ctx, capsys):
    from lsamp import draft_head
    draft_head.main()
    assert "drafts in 8 bits" in capsys.readouterr().out


def test_training_step_with_norms_in_a_graph(ctx):
    """Forward, gradients and the orthogonalised update captured once; each replay is an
    eager step from the same weights."""
    from lsamp.draft_head import DraftHead
    eager = DraftHead(ctx, 128, 600, blocks=1, norm=True, dropout=0.1, seed=8)
    graphed = DraftHead(ctx, 128, 600, blocks=1, norm=True, dropout=0.1, seed=8)
    te, tg = eager.training(64), graphed.training(64)
    for t in (te, tg):
        _batch(t)
        t.launch()
        t.update_orthogonal(0.02, plain_rate=0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tg.launch()
        tg.update_orthogonal(0.02, plain_rate=0.5)
    for step in range(3):
        for t in (te, tg):
            _batch(t, seed=10 + step)
        te.launch()
        te.update_orthogonal(0.02, plain_rate=0.5)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.weights + [eager.head], graphed.weights + [graphed.head]):
            assert torch.equal(a, b), step
