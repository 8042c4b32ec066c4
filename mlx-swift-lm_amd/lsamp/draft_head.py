"""A draft head on the hidden-state operators: trained on a target model's
hidden states, and drawn from by the speculative step.

    x        hidden states of the target model, [rows, hidden]
    block i: x <- x + silu(dropout(x) W_i^T + b_i)
    logits   = x H^T          (H: the vocabulary head, the target's or its own)

Training runs dropout, blocks, the head's cross entropy and every gradient as
prepared calls over fixed buffers (one batch size a plan, graph-capturable);
serving runs the blocks and the logits without dropout and draws with
lsamp_propose, so that the verify step accepts the drafts it would draw itself.

    python -m lsamp.draft_head        # a small head trained on one GPU
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import _ffi
from .api import Context


class DraftHead:
    """Weights of a draft head: `blocks` square layers and a vocabulary head."""

    def __init__(self, ctx: Context, hidden: int, vocab: int, *, blocks: int = 1,
                 dtype: torch.dtype = torch.bfloat16, head: Optional[torch.Tensor] = None,
                 dropout: float = 0.0, seed: int = 0):
        dev = torch.device("cuda", ctx.device)
        g = torch.Generator(device=dev).manual_seed(seed)
        self.ctx, self.hidden, self.vocab, self.dtype = ctx, hidden, vocab, dtype
        self.dropout, self.seed = dropout, seed

        def init(r, c):
            return (torch.randn((r, c), generator=g, device=dev) / c ** 0.5).to(dtype)

        # (blocks start as the identity: their weights are small)
        self.weights: List[torch.Tensor] = [init(hidden, hidden) * 0.1 for _ in range(blocks)]
        self.biases = [torch.zeros(hidden, dtype=dtype, device=dev) for _ in range(blocks)]
        self.head = init(vocab, hidden) if head is None else head

    def training(self, rows: int) -> "Training":
        return Training(self, rows)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """The head's hidden states, as served."""
        for w, b in zip(self.weights, self.biases):
            x = self.ctx.linear(x, w, bias=b, activation="silu", residual=x)
        return x

    def logits(self, x: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return self.ctx.linear(self.forward(x), self.head, out_dtype=dtype)

    def propose(self, x: torch.Tensor, params, **draw) -> torch.Tensor:
        """One draft token a row (`draw`: uniforms or philox_keys)."""
        return self.ctx.propose(self.logits(x), params, **draw)

    def score(self, x: torch.Tensor, targets: torch.Tensor) -> dict:
        """Loss and log-sum-exp of every row's target, without logits."""
        return self.ctx.head_loss(self.forward(x), self.head, targets)


class Training:
    """The prepared calls of one training step of `rows` rows.  Write the batch
    into `x` and `targets` (negative: not trained on) and the rows' share of the
    loss into `d_loss`; `launch()` leaves the losses in `loss` and the gradients
    in `grads`.  Each launch drops other elements."""

    def __init__(self, m: DraftHead, rows: int):
        dev = m.head.device
        c = m.ctx
        self.model, self.rows = m, rows
        self.x = torch.zeros((rows, m.hidden), dtype=m.dtype, device=dev)
        self.targets = torch.full((rows,), -1, dtype=torch.int32, device=dev)
        self.d_loss = torch.full((rows,), 1.0 / rows, device=dev)
        self.step = torch.zeros(1, dtype=torch.int64, device=dev)
        self.calls, back = [], []
        h = self.x
        for i, (w, b) in enumerate(zip(m.weights, m.biases)):
            drop = dict(p=m.dropout, key=m.seed, offset=i << 48, step=self.step)
            d = c.prepare_dropout(h, **drop) if m.dropout else None
            into = d.out if d else h
            f = c.prepare_linear(into, w, bias=b, activation="silu", residual=h, want_pre=True)
            self.calls += ([d] if d else []) + [f]
            back.append((w, into, f, drop))
            h = f.out
        loss = c.prepare_head_loss(h, m.head, self.targets)
        dh = c.prepare_head_loss_backward(self.d_loss, h, m.head, self.targets, lse=loss.lse)
        self.calls += [loss, dh]
        self.loss, self.row_flags = loss.loss, loss.row_flags
        self.grads = {"head": dh.d_weight}
        g = dh.d_x
        for i in reversed(range(len(back))):
            w, into, f, drop = back[i]
            b = c.prepare_linear_backward(g, into, w, pre=f.pre, activation="silu", want_bias=True)
            self.grads[f"weight{i}"], self.grads[f"bias{i}"] = b.d_weight, b.d_bias
            self.calls.append(b)
            if i:  # the gradient of this block's input: through the block, and past it
                through = c.prepare_dropout(b.d_x, residual=g, **drop) if m.dropout else None
                if through is None:  # (p = 0 keeps every element)
                    through = c.prepare_dropout(b.d_x, p=0.0, key=0, residual=g)
                self.calls.append(through)
                g = through.out

    def launch(self) -> None:
        self.step.add_(1)
        for call in self.calls:
            call.launch()

    def update(self, rate: float) -> None:
        """A step of plain gradient descent."""
        m = self.model
        m.head.add_(self.grads["head"], alpha=-rate)
        for i, (w, b) in enumerate(zip(m.weights, m.biases)):
            w.add_(self.grads[f"weight{i}"], alpha=-rate)
            b.add_(self.grads[f"bias{i}"], alpha=-rate)


def main() -> None:
    from . import workloads as W
    ctx = Context(0, max_rows=64, max_vocab=4096)
    m = DraftHead(ctx, 256, 4096, blocks=2, dropout=0.1)
    t = m.training(512)
    g = torch.Generator(device="cuda").manual_seed(1)
    t.targets.copy_(torch.randint(0, 64, (512,), generator=g, device="cuda").int())
    # hidden states that tell the target: a row of a fixed code for each
    code = torch.randn((64, 256), generator=g, device="cuda")
    for step in range(20):
        noise = torch.randn((512, 256), generator=g, device="cuda")
        t.x.copy_(code[t.targets.long()] + 0.3 * noise)
        t.launch()
        t.update(2.0)
        if step % 5 == 4:
            print(f"step {step + 1}: loss {float(t.loss.mean()):.3f}")
    params = W._params([W.resolve_cbv2(temperature=0.0, vocab=4096)] * 8)
    drafts = m.propose(t.x[:8], params, uniforms=torch.zeros(8, device="cuda"))
    print("targets", t.targets[:8].tolist(), "drafts", drafts.tolist())
    ctx.close()


if __name__ == "__main__":
    main()
