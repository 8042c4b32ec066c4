"""The draft head's states: what a quantised head keeps while its source trains on, and the
momenta of updates that are captured."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lsamp.api import Context
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    c = Context(0, max_rows=64, max_vocab=2048)
    yield c
    c.close()


def _batch(t, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t.targets.copy_(torch.randint(0, 500, t.targets.shape, generator=g, device="cuda").int())
    t.x.copy_(torch.randn(t.x.shape, generator=g, device="cuda"))


@pytest.mark.parametrize("orthogonal", [False, True], ids=["plain", "orthogonal"])
def test_a_quantised_head_stays_as_it_was_made(ctx, orthogonal):
    from lsamp.draft_head import DraftHead
    m = DraftHead(ctx, 128, 1000, blocks=2, norm=True, seed=3)
    q = m.quantized()
    t = m.training(64)
    _batch(t)
    x = t.x[:16].clone()
    want = q.logits(x)
    for step in range(2):
        t.launch()
        if orthogonal:
            t.update_orthogonal(0.1, plain_rate=2.0)
        else:
            t.update(2.0)
    assert torch.equal(q.logits(x), want)
    assert not torch.equal(m.quantized().logits(x), want)
    with pytest.raises(TypeError):
        q.quantized()


def _step(t):
    t.launch()
    t.update_orthogonal(0.05, plain_rate=0.5)


def test_the_first_update_is_not_captured(ctx):
    """Its momenta would be cleared by every replay."""
    from lsamp.draft_head import DraftHead
    t = DraftHead(ctx, 64, 500, blocks=1, seed=7).training(16)
    _batch(t)
    t.launch()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="prepare_orthogonal"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            _step(t)
    assert not t.orth


@pytest.mark.parametrize("fast", [False, True], ids=["full", "fast"])
def test_captured_updates_keep_their_momenta(ctx, fast):
    """Replays from the first step on are the eager steps."""
    from lsamp.draft_head import DraftHead
    runs = []
    for graphed in (False, True):
        t = DraftHead(ctx, 128, 600, blocks=2, norm=True, seed=8).training(32)
        t.prepare_orthogonal(fast=fast)
        _batch(t)
        t.launch()
        torch.cuda.synchronize()
        step, g = _step, torch.cuda.CUDAGraph()
        if graphed:
            with torch.cuda.graph(g):
                _step(t)
            step = lambda t, g=g: g.replay()  # noqa: E731
        seen = []
        for i in range(4):
            _batch(t, seed=20 + i)
            step(t)
            torch.cuda.synchronize()
            seen.append([w.clone() for w in t.model.weights + t.momenta])
        runs.append(seen)
    for eager, replayed in zip(*runs):
        assert all(torch.equal(a, b) for a, b in zip(eager, replayed))
    assert float(runs[0][3][-1].norm()) > 1.2 * float(runs[0][0][-1].norm()), "momenta add up"
