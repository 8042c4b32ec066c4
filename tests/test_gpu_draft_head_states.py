"""The draft head's states: what a quantised head keeps while its source trains on."""
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
