"""Masks of several layers and steps under one key (lsamp_dropout), with offsets
that keep their counters apart."""
from __future__ import annotations

import os
import re

import pytest
import torch

import head_common as H

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_example_offsets_keep_layers_apart():
    """Every dropout example in the integration text gives layer L + 1 at one step
    another counter than layer L at any of 1,000 others."""
    text = open(os.path.join(REPO, "INTEGRATION.md")).read()
    found = re.findall(r"p\.offset = ([^;]+);", text) + re.findall(r"dropout\([^\n]*offset=([^\n]+?), r", text)
    assert len(found) == 2
    for expr in found:
        f = eval("lambda layer, step: " + expr.replace("(uint64_t)", ""))
        step_is_added = "step" not in expr
        counters = [f(layer, step) + (step if step_is_added else 0)
                    for layer in range(4) for step in range(1000)]
        assert len(set(counters)) == len(counters), expr


@pytest.mark.gpu
def test_masks_of_layers_and_steps_differ():
    from lsamp.api import Context
    ctx = Context(0, max_rows=4, max_vocab=1024)
    x = torch.ones(16, 256, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    masks = []
    for layer in range(3):
        call = ctx.prepare_dropout(x, p=0.5, key=11, offset=layer << 48, step=step)
        for s in range(3):
            step.fill_(s)
            call.launch()
            kept = (call.out != 0).cpu()
            assert torch.equal(kept, H.philox_keep(16, 256, 0.5, 11, (layer << 48) + s))
            masks.append(kept)
    assert all(not torch.equal(a, b) for i, a in enumerate(masks) for b in masks[:i])
    ctx.close()
