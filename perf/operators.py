"""The operators in front of the logits-to-token stage whose speed is measured: a draft head's
linear blocks, the vocabulary head's loss and their gradients, and the dropout that training them
uses.

A draft head turns a target model's hidden states into drafts: blocks `act(x W^T + b) + x`, then a
vocabulary head whose logits `lsamp_propose` and `lsamp_sample` draw from.  It is trained on the
target's hidden states with dropout and the cross entropy of the vocabulary head.  Serving calls
have a row a stream (1 to some hundreds), training calls a row a token (thousands).

`run` computes each case in plain torch operations, or (`own`) through the library's entry points:
`Context.prepare_linear`, `prepare_linear_backward`, `prepare_head_loss`,
`prepare_head_loss_backward` and `prepare_dropout`.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}

# What a case leaves unsaid.  `train`: the forward pass and its gradients.  `pad`: every matrix is
# a view of rows padded by 8 elements.  linear: [rows, inner] x [outer, inner]; loss: `outer` is the
# vocabulary; dropout: [rows, inner].  `ignored`: the share of rows whose target is ignored.
# `scale`: what the training loop multiplies its loss with.
BASE = dict(train=False, dtype="bf16", pad=False, outer=0, activation="none", softcap=0.0,
            bias=False, residual=False, wide_out=False, ignored=0.0, scale=1.0, p=0.0)


def _case(name, op, rows, inner, **kw):
    return dict(BASE, op=op, rows=rows, inner=inner, **({"name": name} if name else {}), **kw)


def listed():
    return [
        # One stream drafts one token: a block of a draft head.  Nothing but latency and 8 MB.
        _case("block_one_token", "linear", 1, 2048, outer=2048, activation="silu", bias=True,
              residual=True),
        # The logits of a decode batch, for the sampling step: one pass over the head's weights.
        _case("logits_batch", "linear", 64, 2048, outer=151936),
        # A float16 head of odd sizes, a batch of verify windows.
        _case("block_ragged", "linear", 301, 1537, dtype="f16", outer=2053, activation="gelu",
              bias=True, residual=True),
        # A small block trained in float32.
        _case("block_train_f32", "linear", 515, 896, train=True, dtype="f32", outer=1152,
              activation="gelu_tanh", bias=True, residual=True),
        # A block of a large draft head, trained on 8,192 tokens.
        _case("block_train", "linear", 8192, 4096, train=True, outer=4096, activation="silu",
              bias=True, residual=True),
        # Log-probabilities of a few verify windows' tokens, straight from their hidden states.
        _case("score_windows", "loss", 20, 2048, outer=151936),
        # Scoring a long prompt (perplexity): every token's loss.
        _case("score_prompt", "loss", 2048, 4096, outer=128256),
        # A float16 head with a soft cap and a bias over an odd vocabulary, a scaled loss, and a
        # prompt part whose tokens are not trained on.
        _case("head_train_ragged", "loss", 333, 1000, train=True, dtype="f16", outer=40003,
              softcap=30.0, bias=True, ignored=0.25, scale=1024.0),
        # A small vocabulary in float32, a short batch.
        _case("head_train_f32", "loss", 128, 512, train=True, dtype="f32", outer=32000),
        # The head of a large model trained on 4,096 tokens: the largest call.
        _case("head_train", "loss", 4096, 4096, train=True, outer=151936, ignored=0.1),
        # Dropout before a block, a small batch: forward and backward.
        _case("dropout_small", "dropout", 64, 2048, train=True, p=0.1, residual=True),
        # Dropout and residual of a long training batch.
        _case("dropout_large", "dropout", 16384, 8192, train=True, p=0.1, residual=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _odd(rng, low, high):
    """A size of the range: a multiple of 64, of 8, or any number."""
    n, m = _log_int(rng, low, high), rng.choice([64, 64, 8, 1])
    return max(m, n // m * m) if m > 1 else n


def draw(rng):
    op = rng.choice(["linear", "linear", "loss", "loss", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
    train, pad = rng.random() < 0.5, rng.random() < 0.3
    if op == "dropout":
        inner = _odd(rng, 64, 8192)
        rows = _log_int(rng, 1, min(16384, (1 << 27) // inner // (2 if dtype == "f32" else 1)))
        return _case(None, op, rows, inner, train=train, dtype=dtype, pad=pad,
                     p=rng.choice([0.05, 0.1, 0.25, 0.5]), residual=rng.random() < 0.5)
    inner = _odd(rng, 128, 4096)
    if op == "linear":
        outer = rng.choice([_odd(rng, 128, 8192), _odd(rng, 128, 8192), 32000, 151936])
        most = int(1.4e11 / (inner * outer))  # (half of the largest listed block's products)
        rows = _log_int(rng, 1, max(1, min(8192, most)))
        return _case(None, op, rows, inner, train=train, dtype=dtype, pad=pad, outer=outer,
                     activation=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                     bias=rng.random() < 0.7, residual=rng.random() < 0.5,
                     wide_out=not train and rng.random() < 0.2)
    outer = rng.choice([32000, 128256, 151936, _odd(rng, 4000, 262144), _odd(rng, 4000, 262144)])
    most = int(1.2e12 / (inner * outer))  # (half of the largest listed head's products)
    rows = _log_int(rng, 1, max(1, min(4096, most)))
    return _case(None, op, rows, inner, train=train, dtype=dtype, pad=pad, outer=outer,
                 softcap=rng.choice([0.0, 0.0, 30.0]), bias=rng.random() < 0.3,
                 ignored=rng.choice([0.0, 0.25]), scale=1024.0 if dtype == "f16" else 1.0)


# ------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """Hidden states as a norm leaves them, weights as an initialised or trained layer has them.
    A loss row's hidden state leans towards its target's weight row, as a trained head's does."""
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    m, k, n = case["rows"], case["inner"], case["outer"]

    def matrix(r, c, std, more=None):
        t = torch.randn((r, c), generator=g, device=DEVICE)
        t = t.mul_(std) if more is None else t.mul_(std).add_(more)
        if not case["pad"]:
            return t.to(dt)
        wide = torch.zeros((r, c + 8), dtype=dt, device=DEVICE)
        wide[:, :c] = t
        return wide[:, :c]

    s = {"case": case}
    if case["op"] == "dropout":
        s["x"] = matrix(m, k, 1.0)
        s["residual"] = matrix(m, k, 1.0) if case["residual"] else None
        s["d_out"] = matrix(m, k, 0.01) if case["train"] else None
        s["key"] = int(seed) * 0x9E3779B97F4A7C15 % (1 << 64)
        s["offset"] = (int(seed) % 1000) << 20
        return s
    s["weight"] = matrix(n, k, (2.0 if case["op"] == "loss" else 1.0) / math.sqrt(k))
    s["bias"] = (torch.randn(n, generator=g, device=DEVICE) * 0.1).to(dt) if case["bias"] else None
    if case["op"] == "linear":
        s["x"] = matrix(m, k, 1.0)
        s["residual"] = matrix(m, n, 1.0) if case["residual"] else None
        s["d_out"] = matrix(m, n, 0.01) if case["train"] else None
        return s
    # token frequencies fall as 1 / (rank + 10)
    u = torch.rand(m, generator=g, device=DEVICE, dtype=torch.float64)
    rank = (10.0 * torch.exp(u * math.log((n + 10.0) / 10.0)) - 10.0).long().clamp_(0, n - 1)
    targets = rank * 7919 % n
    lean = torch.rand((m, 1), generator=g, device=DEVICE) * 2.0
    s["x"] = matrix(m, k, 1.0, lean * s["weight"][targets].float())
    ignored = torch.rand(m, generator=g, device=DEVICE) < case["ignored"]
    s["targets"] = torch.where(ignored, -100, targets).to(torch.int32)
    if case["train"]:
        kept = (~ignored).sum().clamp(min=1).float()
        s["d_loss"] = (case["scale"] / kept).expand(m).contiguous()  # the mean over trained tokens
    return s


_context = None


def _calls(case, s):
    """The prepared calls that a program keeps between passes."""
    global _context
    if _context is None:
        sys.path.insert(1, os.path.join(os.getcwd(), "mlx-swift-lm_amd"))
        from lsamp.api import Context
        _context = Context(0, max_rows=1, max_vocab=1024)
    c = _context
    if case["op"] == "dropout":
        kw = dict(p=case["p"], key=s["key"], offset=s["offset"])
        calls = [c.prepare_dropout(s["x"], residual=s["residual"], **kw)]
        if case["train"]:
            calls.append(c.prepare_dropout(s["d_out"], **kw))
    elif case["op"] == "linear":
        act = case["activation"]
        kept = case["train"] and act != "none"  # the backward pass reads the pre-activations
        calls = [c.prepare_linear(s["x"], s["weight"], bias=s["bias"], residual=s["residual"],
                                  activation=act, want_pre=kept,
                                  out_dtype=torch.float32 if case["wide_out"] else None)]
        if case["train"]:
            calls.append(c.prepare_linear_backward(s["d_out"], s["x"], s["weight"],
                                                   pre=calls[0].pre, activation=act,
                                                   want_bias=case["bias"]))
    else:
        kw = dict(bias=s["bias"], softcap=case["softcap"])
        calls = [c.prepare_head_loss(s["x"], s["weight"], s["targets"], **kw)]
        if case["train"]:
            calls.append(c.prepare_head_loss_backward(s["d_loss"], s["x"], s["weight"],
                                                      s["targets"], lse=calls[0].lse,
                                                      want_bias=case["bias"], **kw))
    return calls


def prepare(case, seed):
    case = dict(BASE, **case)
    s = _inputs(case, seed)
    if own:
        s["calls"] = _calls(case, s)
    return s


# ----------------------------------------------------------------------------------- plain form
def _activation(name, z):
    """act(z) and act'(z)."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return z * sig, sig * (1 + z * (1 - sig))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        d = 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
        return 0.5 * z * (1 + t), d
    return z, torch.ones_like(z)


def _linear(s, case, to):
    """The block and its gradients, in the type `to`."""
    x, w = s["x"].to(to), s["weight"].to(to)
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].to(to)
    y, slope = _activation(case["activation"], z)
    if s["residual"] is not None:
        y = y + s["residual"].to(to)
    out = {"out": y}
    if case["train"]:
        dz = s["d_out"].to(to) * slope
        out["d_x"], out["d_weight"] = dz @ w, dz.t() @ x
        if s["bias"] is not None:
            out["d_bias"] = dz.sum(0)
    return out


def _loss(s, case, to):
    """The loss of every row from its whole row of logits, and the gradients of its weighted sum."""
    x, w = s["x"].to(to), s["weight"].to(to)
    z = x @ w.t()
    if s["bias"] is not None:
        z += s["bias"].to(to)
    cap = case["softcap"]
    if cap:
        z = cap * torch.tanh(z / cap)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    t = s["targets"].long()
    kept = t >= 0
    at = t.clamp(min=0)[:, None]
    loss = torch.where(kept, (lse - z.gather(1, at))[:, 0], torch.zeros((), dtype=to, device=t.device))
    out = {"loss": loss, "lse": lse[:, 0]}
    if case["train"]:
        d = e.div_(total)
        d.scatter_add_(1, at, torch.full_like(lse, -1.0))
        d *= (s["d_loss"].to(to) * kept)[:, None]
        if cap:
            d *= 1 - (z / cap) ** 2
        out["d_x"], out["d_weight"] = d @ w, d.t() @ x
        if s["bias"] is not None:
            out["d_bias"] = d.sum(0)
    return out


def _philox(c0, c1, c2, c3, key):
    """Philox4x32-10 of counters held in int64 tensors: products wrap to their low 64 bits."""
    low = 0xFFFFFFFF
    k0, k1 = key & low, key >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _dropout(s, case):
    """Eight elements of a row share one draw of 128 bits, 16 bits each; an element is kept where
    its bits are at least round(p 2^16)."""
    m, k = s["x"].shape
    groups = (k + 7) // 8
    c0 = torch.arange(groups, device=DEVICE)[None, :].expand(m, groups)
    c1 = torch.arange(m, device=DEVICE)[:, None].expand(m, groups)
    c2, c3 = (torch.full_like(c0, v) for v in (s["offset"] & 0xFFFFFFFF, s["offset"] >> 32))
    words = torch.stack(_philox(c0, c1, c2, c3, s["key"]), -1)
    bits = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(m, groups * 8)[:, :k]
    cut = round(case["p"] * 65536)
    scale = (bits >= cut).float() * (65536.0 / (65536 - cut))
    y = s["x"].float() * scale
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"out": y}
    if case["train"]:
        out["d_x"] = s["d_out"].float() * scale
    return out


def run(s):
    case = s["case"]
    if own:
        out = {}
        for call in s["calls"]:
            call.launch()
            out.update(call.outputs())
        return {k: out[k] for k in ("out", "loss", "lse", "d_x", "d_weight", "d_bias") if k in out
                } if case["op"] != "dropout" else dict(
            {"out": s["calls"][0].out}, **({"d_x": s["calls"][1].out} if case["train"] else {}))
    if case["op"] == "dropout":
        out = _dropout(s, case)
    else:
        out = (_linear if case["op"] == "linear" else _loss)(s, case, torch.float32)
    wide = ("loss", "lse") + (("out",) if case["wide_out"] else ())
    return {k: v if k in wide else v.to(DTYPES[case["dtype"]]) for k, v in out.items()}


# ----------------------------------------------------------------------------------------- work
def work(case):
    c = dict(BASE, **case)
    m, k, n, e = c["rows"], c["inner"], c["outer"], SIZE[c["dtype"]]
    if c["op"] == "dropout":
        one = m * k
        moved = one * e * ((3 if c["residual"] else 2) + (2 if c["train"] else 0))
        return {"bytes": moved, "flops": one * (3 if c["train"] else 2)}
    passes = 3 if c["train"] else 1  # the product, and with gradients two more
    flops = 2 * m * n * k * passes
    moved = (m * k + n * k) * e * (2 if c["train"] else 1)
    moved += n * e * c["bias"] * (2 if c["train"] else 1)
    if c["op"] == "linear":
        moved += m * n * (4 if c["wide_out"] else e) + m * n * e * (c["residual"] + c["train"])
    else:
        moved += m * 4 * (4 if c["train"] else 3)
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------------------- exact
def _exact_act(name, z):
    """act(z) and its derivative in 64 bits, by other forms than the plain one's."""
    if name == "relu":
        return torch.maximum(z, torch.zeros_like(z)), torch.heaviside(z, torch.zeros_like(z))
    if name == "silu":
        sig = 0.5 + 0.5 * torch.tanh(0.5 * z)
        y = z * sig
        return y, y + sig - y * sig
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-(z ** 2) / 2) * 0.3989422804014327
    if name == "gelu_tanh":
        a, b = 2 * math.sqrt(2 / math.pi), 0.044715
        sig = 1 / (1 + torch.exp(-a * z * (1 + b * z ** 2)))  # (1 + tanh(u)) / 2 = sigmoid(2 u)
        return z * sig, sig + z * sig * (1 - sig) * a * (1 + 3 * b * z ** 2)
    return z, torch.ones_like(z)


def _exact_keep(m, k, p, key, offset):
    """The kept elements, from Philox's definition on unsigned 64-bit integers."""
    u64, low = np.uint64, np.uint64(0xFFFFFFFF)
    g = (k + 7) // 8
    ctr = [np.tile(np.arange(g, dtype=u64), m), np.repeat(np.arange(m, dtype=u64), g),
           np.full(m * g, offset % (1 << 32), u64), np.full(m * g, offset >> 32, u64)]
    keys = [key % (1 << 32), key >> 32]
    for _ in range(10):
        p0, p1 = ctr[0] * u64(0xD2511F53), ctr[2] * u64(0xCD9E8D57)
        ctr = [(p1 >> u64(32)) ^ ctr[1] ^ u64(keys[0]), p1 & low,
               (p0 >> u64(32)) ^ ctr[3] ^ u64(keys[1]), p0 & low]
        keys = [(keys[0] + 0x9E3779B9) % (1 << 32), (keys[1] + 0xBB67AE85) % (1 << 32)]
    words = np.stack([c.astype("<u4") for c in ctr], 1)
    return words.view("<u2").reshape(m, g * 8)[:, :k] >= int(round(p * 65536))


def exact(case, seed):
    c = dict(BASE, **case)
    s = _inputs(c, seed)
    f64 = torch.float64
    if c["op"] == "dropout":
        m, k = s["x"].shape
        keep = torch.from_numpy(_exact_keep(m, k, c["p"], s["key"], s["offset"])).to(DEVICE)
        scale = 65536.0 / (65536.0 - round(c["p"] * 65536))
        zero = torch.zeros((), dtype=f64, device=DEVICE)
        y = torch.where(keep, s["x"].to(f64) * scale, zero)
        out = {"out": y if s["residual"] is None else s["residual"].to(f64) + y}
        if c["train"]:
            out["d_x"] = torch.where(keep, s["d_out"].to(f64) * scale, zero)
        return out
    x, w = s["x"].to(f64), s["weight"].to(f64)
    if c["op"] == "linear":
        wt = w.t().contiguous()
        z = x @ wt if s["bias"] is None else torch.addmm(s["bias"].to(f64), x, wt)
        y, slope = _exact_act(c["activation"], z)
        out = {"out": y if s["residual"] is None else y + s["residual"].to(f64)}
        if c["train"]:
            dz = slope * s["d_out"].to(f64)
            out["d_x"], out["d_weight"] = dz @ w, dz.t().contiguous() @ x
            if s["bias"] is not None:
                out["d_bias"] = torch.ones(c["rows"], dtype=f64, device=DEVICE) @ dz
        return out
    # the loss over blocks of rows, each row's own softmax
    m, cap = c["rows"], c["softcap"]
    loss, lse, d_x = [], [], []
    d_w = torch.zeros_like(w) if c["train"] else None
    d_b = torch.zeros(c["outer"], dtype=f64, device=DEVICE) if c["train"] and c["bias"] else None
    for lo in range(0, m, 1024):
        xs, t = x[lo:lo + 1024], s["targets"][lo:lo + 1024].long()
        z = xs @ w.t().contiguous()
        if s["bias"] is not None:
            z += s["bias"].to(f64)
        slope = None
        if cap:
            z = torch.tanh(z / cap)
            slope = 1 - z * z
            z = z * cap
        whole = torch.logsumexp(z, 1)
        row = torch.arange(len(t), device=DEVICE)
        ok = t >= 0
        loss.append(torch.where(ok, whole - z[row, t.clamp(min=0)], torch.zeros_like(whole)))
        lse.append(whole)
        if c["train"]:
            g = torch.softmax(z, 1)
            g[row, t.clamp(min=0)] -= 1
            g *= torch.where(ok, s["d_loss"][lo:lo + 1024].to(f64), torch.zeros_like(whole))[:, None]
            g = g if slope is None else g * slope
            d_x.append(g @ w)
            d_w += g.t().contiguous() @ xs
            if d_b is not None:
                d_b += g.sum(0)
    out = {"loss": torch.cat(loss), "lse": torch.cat(lse)}
    if c["train"]:
        out.update(d_x=torch.cat(d_x), d_weight=d_w)
        if d_b is not None:
            out["d_bias"] = d_b
    return out
