"""A draft head on the hidden-state operators: trained on a target model's
hidden states, and drawn from by the speculative step.

    x        hidden states of the target model, [rows, hidden]
    block i: x <- x + silu(dropout(norm_i(x)) W_i^T + b_i)
    logits   = norm(x) H^T    (H: the vocabulary head, the target's or its own)

(the norms, layer norms with a weight and a bias, only with `norm`.)

Training runs norms, dropout, blocks, the head's cross entropy and every gradient
as prepared calls over fixed buffers (one batch size a plan, graph-capturable), and
updates plainly or with orthogonalised momenta of the blocks' matrices; serving
runs the blocks and the logits without dropout, in the weights' type or in 8-bit
integers (`quantized`), and draws with lsamp_propose, so that the verify step
accepts the drafts it would draw itself.

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
                 dropout: float = 0.0, norm: bool = False, seed: int = 0):
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
        # one in front of every block, and one in front of the vocabulary head
        self.norms = [(torch.ones(hidden, dtype=dtype, device=dev),
                       torch.zeros(hidden, dtype=dtype, device=dev))
                      for _ in range(blocks + 1)] if norm else []

    def training(self, rows: int) -> "Training":
        return Training(self, rows)

    def quantized(self) -> "Int8DraftHead":
        """The same head served with 8-bit products (its weights as they are now)."""
        return Int8DraftHead(self)

    def _norm(self, i: int, x: torch.Tensor) -> torch.Tensor:
        if not self.norms:
            return x
        w, b = self.norms[i]
        return self.ctx.layer_norm(x, weight=w, bias=b)

    def _block(self, i: int, x: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
        return self.ctx.linear(x, self.weights[i], bias=self.biases[i], activation="silu",
                               residual=residual)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """The head's hidden states, as served."""
        for i in range(len(self.biases)):
            x = self._block(i, self._norm(i, x), x)
        return self._norm(len(self.biases), x)

    def logits(self, x: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return self.ctx.linear(self.forward(x), self.head, out_dtype=dtype)

    def propose(self, x: torch.Tensor, params, **draw) -> torch.Tensor:
        """One draft token a row (`draw`: uniforms or philox_keys)."""
        return self.ctx.propose(self.logits(x), params, **draw)

    def score(self, x: torch.Tensor, targets: torch.Tensor) -> dict:
        """Loss and log-sum-exp of every row's target, without logits."""
        return self.ctx.head_loss(self.forward(x), self.head, targets)


class Int8DraftHead(DraftHead):
    """A draft head whose matrices are 8-bit integers with a scale for each output,
    and whose tokens are quantised as they come.  Serves; is not trained."""

    def __init__(self, m: DraftHead):
        self.ctx, self.hidden, self.vocab, self.dtype = m.ctx, m.hidden, m.vocab, m.dtype
        # (copies: training goes on in the vectors of the head that it was made from)
        self.biases = [b.clone() for b in m.biases]
        self.norms = [(w.clone(), b.clone()) for w, b in m.norms]
        self.weights = [self.ctx.quantize_rows(w) for w in m.weights]
        self.head = self.ctx.quantize_rows(m.head)

    def _block(self, i: int, x: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
        return self.ctx.linear_int8(x, *self.weights[i], bias=self.biases[i], activation="silu",
                                    residual=residual)

    def logits(self, x: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return self.ctx.linear_int8(self.forward(x), *self.head, out_dtype=dtype)

    def quantized(self) -> "Int8DraftHead":
        raise TypeError("a quantised head is one already")

    def training(self, rows: int) -> "Training":
        raise TypeError("a quantised head is not trained: train the one it was made from")

    def score(self, x: torch.Tensor, targets: torch.Tensor) -> dict:
        raise TypeError("a quantised head has no loss: score with the one it was made from")


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
        self.momenta, self.orth = [], []
        h = self.x

        def norm(i):
            if not m.norms:
                return None
            w, b = m.norms[i]
            n = c.prepare_layer_norm(h, weight=w, bias=b, want_stats=True)
            self.calls.append(n)
            return n, h, w

        def norm_gradient(i, n, d, past, want_x=True):
            """The gradient at a norm's input, with the one that comes past it."""
            n, x, w = n
            b = c.prepare_layer_norm_backward(d, x, mean=n.mean, rstd=n.rstd, weight=w,
                                              residual=past, want_x=want_x, want_bias=True)
            self.grads[f"norm_weight{i}"], self.grads[f"norm_bias{i}"] = b.d_weight, b.d_bias
            self.calls.append(b)
            return b.d_x

        for i, (w, b) in enumerate(zip(m.weights, m.biases)):
            drop = dict(p=m.dropout, key=m.seed, offset=i << 48, step=self.step)
            n = norm(i)
            into = n[0].out if n else h
            d = c.prepare_dropout(into, **drop) if m.dropout else None
            into = d.out if d else into
            f = c.prepare_linear(into, w, bias=b, activation="silu", residual=h, want_pre=True)
            self.calls += ([d] if d else []) + [f]
            back.append((w, into, f, drop, n))
            h = f.out
        last = norm(len(back))
        h = last[0].out if last else h
        loss = c.prepare_head_loss(h, m.head, self.targets)
        dh = c.prepare_head_loss_backward(self.d_loss, h, m.head, self.targets, lse=loss.lse)
        self.calls += [loss, dh]
        self.loss, self.row_flags = loss.loss, loss.row_flags
        self.grads = {"head": dh.d_weight}
        g = dh.d_x
        if last:
            g = norm_gradient(len(back), last, g, None)
        for i in reversed(range(len(back))):
            w, into, f, drop, n = back[i]
            b = c.prepare_linear_backward(g, into, w, pre=f.pre, activation="silu", want_bias=True)
            self.grads[f"weight{i}"], self.grads[f"bias{i}"] = b.d_weight, b.d_bias
            self.calls.append(b)
            if n:  # through the dropout and the norm, and past them
                d = b.d_x
                if m.dropout:
                    through = c.prepare_dropout(d, **drop)
                    self.calls.append(through)
                    d = through.out
                g = norm_gradient(i, n, d, g if i else None, want_x=i > 0)
            elif i:  # the gradient of this block's input: through the block, and past it
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
        for i, w in enumerate(self.model.weights):
            w.add_(self.grads[f"weight{i}"], alpha=-rate)
        self._plain(rate)

    def _plain(self, rate: float) -> None:
        m = self.model
        m.head.add_(self.grads["head"], alpha=-rate)
        for i, b in enumerate(m.biases):
            b.add_(self.grads[f"bias{i}"], alpha=-rate)
        for i, (w, b) in enumerate(m.norms):
            w.add_(self.grads[f"norm_weight{i}"], alpha=-rate)
            b.add_(self.grads[f"norm_bias{i}"], alpha=-rate)

    def prepare_orthogonal(self, *, fast: bool = False) -> None:
        """The momenta of update_orthogonal, zero, and its calls (`fast`: as
        Context.prepare_orthogonalize has it).  The first update makes them; one that is
        captured into a graph, where every replay would clear them, needs them made
        before."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("momenta are made outside a capture: call prepare_orthogonal before")
        m = self.model
        self.momenta = [torch.zeros(w.shape, device=w.device) for w in m.weights]
        self.nesterov = [torch.empty_like(v) for v in self.momenta]
        self.orth = [m.ctx.prepare_orthogonalize(v, base=w, out=w, fast=fast)
                     for v, w in zip(self.nesterov, m.weights)]

    def update_orthogonal(self, rate: float, *, plain_rate: float, momentum: float = 0.95,
                          decay: float = 0.0) -> None:
        """A step with orthogonalised momenta (Muon's) of the blocks' matrices:
            M <- momentum M + gradient
            W <- (1 - rate decay) W - rate orth(gradient + momentum M)
        and plain descent of the rest at `plain_rate`."""
        m = self.model
        if not self.orth and m.weights:
            self.prepare_orthogonal()
        for i, call in enumerate(self.orth):
            grad = self.grads[f"weight{i}"].float()
            self.momenta[i].mul_(momentum).add_(grad)
            torch.add(grad, self.momenta[i], alpha=momentum, out=self.nesterov[i])
            call.weigh(scale=-rate, keep=1.0 - rate * decay)
            call.launch()
        self._plain(plain_rate)


def main() -> None:
    from . import workloads as W
    ctx = Context(0, max_rows=64, max_vocab=4096)
    m = DraftHead(ctx, 256, 4096, blocks=2, dropout=0.1, norm=True)
    t = m.training(512)
    g = torch.Generator(device="cuda").manual_seed(1)
    t.targets.copy_(torch.randint(0, 64, (512,), generator=g, device="cuda").int())
    # hidden states that tell the target: a row of a fixed code for each
    code = torch.randn((64, 256), generator=g, device="cuda")
    for step in range(20):
        noise = torch.randn((512, 256), generator=g, device="cuda")
        t.x.copy_(code[t.targets.long()] + 0.3 * noise)
        t.launch()
        t.update_orthogonal(0.02, plain_rate=2.0)
        if step % 5 == 4:
            print(f"step {step + 1}: loss {float(t.loss.mean()):.3f}")
    params = W._params([W.resolve_cbv2(temperature=0.0, vocab=4096)] * 8)
    print("targets", t.targets[:8].tolist())
    for name, served in (("drafts", m), ("drafts in 8 bits", m.quantized())):
        drafts = served.propose(t.x[:8], params, uniforms=torch.zeros(8, device="cuda"))
        print(name, drafts.tolist())
    ctx.close()


if __name__ == "__main__":
    main()
