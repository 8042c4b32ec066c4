"""More operators of a draft head whose speed is measured: the layer norm of its blocks and its
gradients, blocks and vocabulary head served in 8-bit integers, and the orthogonalised update that
trains the blocks' matrices.

Serving calls have a row a stream (1 to some hundreds), training calls and prompts a row a token
(thousands).  An update is a call a matrix, or one for a stack of matrices of one shape.

`run` computes each case in plain torch operations, or (`own`) through the library's entry points:
`Context.prepare_layer_norm`, `prepare_layer_norm_backward`, `prepare_quantize_rows`,
`prepare_linear_int8` and `prepare_orthogonalize`.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}

EPS = 1e-5  # of the norm
# The quintic of the Newton-Schulz steps, and what is added to the norm of an update.
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
TINY = 1e-7

# What a case leaves unsaid.  `train`: the forward pass and its gradients.  `pad`: every matrix is
# a view of rows padded by 8 elements.  norm and quantize: [rows, inner]; int8: [rows, inner] x
# [outer, inner]; orth: `batch` matrices [rows, inner].  `given`: x comes quantised.  `weighted`: a
# norm has a weight and a bias.  `update`: out = 0.99 base - 0.02 orth(x), else orth(x).
BASE = dict(train=False, dtype="bf16", pad=False, outer=0, activation="none", bias=False,
            residual=False, wide_out=False, given=False, weighted=True, batch=1, steps=5,
            update=False, wide_in=False)


def _case(name, op, rows, inner, **kw):
    return dict(BASE, op=op, rows=rows, inner=inner, **({"name": name} if name else {}), **kw)


def listed():
    return [
        # One stream's token in front of a block: latency.
        _case("norm_one_token", "norm", 1, 2048),
        # A small float16 batch of odd sizes, trained.
        _case("norm_train_ragged", "norm", 301, 1537, dtype="f16", train=True, residual=True),
        # The norm of a block trained on 16,384 tokens, its skip path's gradient added.
        _case("norm_train", "norm", 16384, 4096, train=True, residual=True),
        # A decode batch's hidden states to 8 bits, for products that share them.
        _case("quantize_batch", "quantize", 64, 4096),
        # A vocabulary head's weights to 8 bits: once, when a model is loaded.
        _case("quantize_head", "quantize", 151936, 2048),
        # One stream drafts one token: a block of a draft head in 8 bits.
        _case("int8_one_token", "int8", 1, 2048, outer=2048, activation="silu", bias=True,
              residual=True),
        # The logits of a decode batch, for the sampling step: one pass over the head's bytes.
        _case("int8_logits_batch", "int8", 64, 2048, outer=151936),
        # A float16 head of odd sizes, a batch of verify windows.
        _case("int8_ragged", "int8", 301, 1537, dtype="f16", outer=2053, activation="gelu",
              bias=True, residual=True),
        # A block over a long prompt.
        _case("int8_prompt", "int8", 8192, 4096, outer=4096, activation="silu", bias=True,
              residual=True),
        # The blocks of a small head, updated in float32 in one call.
        _case("orth_small_f32", "orth", 256, 256, dtype="f32", batch=4, update=True),
        # Two wide matrices of odd sizes: float32 momentum, the orthogonal factor in bfloat16.
        _case("orth_ragged", "orth", 515, 1157, wide_in=True, batch=2),
        # A block's matrix of a large draft head: the largest call.
        _case("orth_large", "orth", 4096, 4096, update=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _odd(rng, low, high):
    """A size of the range: a multiple of 64, of 8, or any number."""
    n, m = _log_int(rng, low, high), rng.choice([64, 64, 8, 1])
    return max(m, n // m * m) if m > 1 else n


def draw(rng):
    op = rng.choice(["norm", "norm", "quantize", "int8", "int8", "int8", "orth", "orth"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
    pad = rng.random() < 0.3
    if op in ("norm", "quantize"):
        inner = _odd(rng, 64, 16384)
        most = (1 << 26) // inner // (2 if dtype == "f32" else 1)
        rows = _log_int(rng, 1, min(32768, most))
        if op == "quantize":
            return _case(None, op, rows, inner, dtype=dtype, pad=pad)
        return _case(None, op, rows, inner, train=rng.random() < 0.6, dtype=dtype, pad=pad,
                     residual=rng.random() < 0.5, weighted=rng.random() < 0.8)
    if op == "int8":
        inner = _odd(rng, 128, 8192)
        outer = rng.choice([_odd(rng, 128, 8192), _odd(rng, 128, 8192), 32000, 151936])
        most = int(1.3e11 / (inner * outer))  # (the products of the largest listed block)
        rows = _log_int(rng, 1, max(1, min(8192, most)))
        return _case(None, op, rows, inner, dtype=dtype, pad=pad, outer=outer,
                     activation=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                     bias=rng.random() < 0.7, residual=rng.random() < 0.5,
                     wide_out=rng.random() < 0.2, given=rng.random() < 0.25)
    rows, inner = _odd(rng, 48, 4096), _odd(rng, 48, 4096)
    small = min(rows, inner)
    most = int(1e11 / (4.0 * small * rows * inner))  # (well below the largest listed update)
    while most < 1:
        rows, inner = (rows + 1) // 2, (inner + 1) // 2
        most = int(1e11 / (4.0 * min(rows, inner) * rows * inner))
    return _case(None, op, rows, inner, dtype=rng.choice(["bf16", "bf16", "bf16", "f16", "f32"]),
                 pad=pad, batch=_log_int(rng, 1, min(16, most)), steps=rng.choice([5, 5, 3, 6]),
                 update=rng.random() < 0.7, wide_in=rng.random() < 0.4)


# ------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """Hidden states as a residual stream has them: rows of different size and offset, some columns
    much larger.  Momenta as training leaves them: a falling spectrum above noise."""
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    m, k, n = case["rows"], case["inner"], case["outer"]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    def view(t, to=dt):
        """`t` as a user holds it: of its type, with padded rows where the case says so."""
        if not case["pad"]:
            return t.to(to)
        wide = torch.zeros(t.shape[:-1] + (t.shape[-1] + 8,), dtype=to, device=DEVICE)
        wide[..., :t.shape[-1]] = t
        return wide[..., :t.shape[-1]]

    def hidden(rows, cols):
        t = randn(rows, cols)
        t[:, ::97] *= 6.0
        return t.mul_(0.5 + torch.rand((rows, 1), generator=g, device=DEVICE)).add_(
            0.2 * randn(rows, 1))

    s = {"case": case}
    if case["op"] == "norm":
        s["x"] = view(hidden(m, k))
        s["weight"] = (1.0 + 0.1 * randn(k)).to(dt) if case["weighted"] else None
        s["bias"] = (0.1 * randn(k)).to(dt) if case["weighted"] else None
        if case["train"]:
            s["d_out"] = view(0.01 * randn(m, k))
            s["residual"] = view(0.01 * randn(m, k)) if case["residual"] else None
    elif case["op"] == "quantize":
        s["x"] = view(hidden(m, k))
    elif case["op"] == "int8":
        s["weight"], s["weight_scale"] = _quantized(randn(n, k).div_(math.sqrt(k)))
        s["weight"] = view(s["weight"], torch.int8)
        x, s["x_scale"] = hidden(m, k).to(dt), None
        if case["given"]:
            x, s["x_scale"] = _quantized(x)
        s["x"] = view(x, x.dtype)
        s["bias"] = (0.1 * randn(n)).to(dt) if case["bias"] else None
        s["residual"] = view(randn(m, n)) if case["residual"] else None
    else:
        b, r = case["batch"], max(1, min(m, k) // 2)
        fall = 1.0 / (torch.arange(r, device=DEVICE) + 4.0)
        x = (randn(b, m, r) * fall) @ randn(b, r, k)
        x = x.add_(randn(b, m, k), alpha=0.02).mul_(1e-4)
        s["x"] = view(x, torch.float32 if case["wide_in"] else dt)
        s["base"] = view(randn(b, m, k) / math.sqrt(k)) if case["update"] else None
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
    if case["op"] == "norm":
        calls = [c.prepare_layer_norm(s["x"], weight=s["weight"], bias=s["bias"], eps=EPS,
                                      want_stats=case["train"])]
        if case["train"]:
            calls.append(c.prepare_layer_norm_backward(
                s["d_out"], s["x"], mean=calls[0].mean, rstd=calls[0].rstd, weight=s["weight"],
                residual=s["residual"], want_weight=case["weighted"],
                want_bias=case["weighted"]))
        return calls
    if case["op"] == "quantize":
        return [c.prepare_quantize_rows(s["x"])]
    if case["op"] == "int8":
        return [c.prepare_linear_int8(s["x"], s["weight"], s["weight_scale"], x_scale=s["x_scale"],
                                      bias=s["bias"], residual=s["residual"],
                                      activation=case["activation"],
                                      out_dtype=DTYPES["f32" if case["wide_out"]
                                                       else case["dtype"]])]
    return [c.prepare_orthogonalize(s["x"], steps=case["steps"], coefficients=COEFFICIENTS,
                                    eps=TINY, base=s["base"],
                                    scale=-0.02 if case["update"] else 1.0,
                                    keep=0.99 if case["update"] else 0.0,
                                    out_dtype=DTYPES[case["dtype"]])]


def prepare(case, seed):
    case = dict(BASE, **case)
    s = _inputs(case, seed)
    if own:
        s["calls"] = _calls(case, s)
    return s


# ----------------------------------------------------------------------------------- plain form
def _norm(s, case):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    xh = centred * rstd
    y = xh
    if s["weight"] is not None:
        y = xh * s["weight"].float() + s["bias"].float()
    out = {"out": y}
    if case["train"]:
        d = s["d_out"].float()
        g = d if s["weight"] is None else d * s["weight"].float()
        d_x = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        out["d_x"] = d_x if s["residual"] is None else d_x + s["residual"].float()
        if s["weight"] is not None:
            out["d_weight"], out["d_bias"] = (d * xh).sum(0), d.sum(0)
    return out


def _quantized(x):
    """Whole numbers up to 127 and a float32 scale for each row; the nearest one to the exact
    quotient, hence 64 bits."""
    scale = (x.abs().amax(1).float() / 127.0).clamp(min=2.0 ** -126)
    return (x.double() / scale.double()[:, None]).round().clamp(-127, 127).to(torch.int8), scale


def _activation(name, z):
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _int8(s, case):
    q, scale = (s["x"], s["x_scale"]) if case["given"] else _quantized(s["x"])
    z = q.float() @ s["weight"].float().t()
    z = z * (scale[:, None] * s["weight_scale"])
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _activation(case["activation"], z)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"out": y}


def _orth(s, case):
    a, b, c = COEFFICIENTS
    x = s["x"].float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / ((x * x).sum((1, 2), keepdim=True).sqrt() + TINY)
    for _ in range(case["steps"]):
        p = x @ x.transpose(1, 2)
        x = a * x + (b * p + c * (p @ p)) @ x
    if tall:
        x = x.transpose(1, 2)
    if s["base"] is not None:
        x = 0.99 * s["base"].float() - 0.02 * x
    return {"out": x.contiguous()}


def run(s):
    case = s["case"]
    if own:
        out = {}
        for call in s["calls"]:
            call.launch()
            out.update(call.outputs())
        return {k: out[k] for k in ("out", "q", "scale", "d_x", "d_weight", "d_bias") if k in out}
    if case["op"] == "quantize":
        return dict(zip(("q", "scale"), _quantized(s["x"])))
    out = {"norm": _norm, "int8": _int8, "orth": _orth}[case["op"]](s, case)
    dt = torch.float32 if case["wide_out"] else DTYPES[case["dtype"]]
    return {k: v.to(dt) for k, v in out.items()}


# ----------------------------------------------------------------------------------------- work
def work(case):
    c = dict(BASE, **case)
    m, k, n, e = c["rows"], c["inner"], c["outer"], SIZE[c["dtype"]]
    if c["op"] == "norm":
        arrays = 2 + (2 + c["residual"] if c["train"] else 0)
        vectors = c["weighted"] * (4 if c["train"] else 2)
        return {"bytes": (arrays * m + vectors) * k * e, "flops": m * k * (22 if c["train"] else 8)}
    if c["op"] == "quantize":
        return {"bytes": m * k * (e + 1) + 4 * m, "flops": 3 * m * k}
    if c["op"] == "int8":
        moved = m * k * (1 if c["given"] else e) + n * k + 4 * n + c["bias"] * n * e
        moved += m * n * ((4 if c["wide_out"] else e) + c["residual"] * e)
        return {"bytes": moved, "flops": 2 * m * n * k}
    small, large = min(m, k), max(m, k)
    # (both products of a matrix with its own transpose are symmetric: half of each)
    flops = c["steps"] * (3 * small * small * large + small ** 3)
    return {"bytes": c["batch"] * m * k * ((4 if c["wide_in"] else e) + e * (1 + c["update"])),
            "flops": c["batch"] * flops}


# ---------------------------------------------------------------------------------------- exact
def _exact_act(name, z):
    """The activations in 64 bits, by other forms than the plain one's."""
    if name == "relu":
        return torch.maximum(z, torch.zeros_like(z))
    if name == "silu":
        return z * (0.5 + 0.5 * torch.tanh(0.5 * z))
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
    if name == "gelu_tanh":
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * z * (1 + 0.044715 * z ** 2)))
    return z


def _exact_norm(c, s):
    """Blocks of rows; the gradient as rstd (I - 1 1^T / n - xh xh^T / n) g."""
    f64, out, d_x = torch.float64, [], []
    k = c["inner"]
    one = torch.ones(k, dtype=f64, device=DEVICE)
    w = one if s["weight"] is None else s["weight"].to(f64)
    b = 0 * one if s["bias"] is None else s["bias"].to(f64)
    d_w, d_b = 0 * one, 0 * one
    for lo in range(0, c["rows"], 4096):
        x = s["x"][lo:lo + 4096].to(f64)
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        xh = (x - mean) / torch.sqrt(var + EPS)
        out.append(torch.addcmul(b, xh, w))
        if c["train"]:
            d = s["d_out"][lo:lo + 4096].to(f64)
            g = d * w
            along = torch.linalg.vecdot(xh, g)
            t = g - (g @ one)[:, None] / k - xh * along[:, None] / k
            t = t / torch.sqrt(var + EPS)
            if s["residual"] is not None:
                t += s["residual"][lo:lo + 4096].to(f64)
            d_x.append(t)
            d_w += torch.linalg.vecdot(d, xh, dim=0)
            d_b += d.sum(0)
    r = {"out": torch.cat(out)}
    if c["train"]:
        r["d_x"] = torch.cat(d_x)
        if s["weight"] is not None:
            r["d_weight"], r["d_bias"] = d_w, d_b
    return r


def _exact_quantized(x):
    """floor of twice the quotient decides between the two neighbours; ties go to the even one."""
    top = torch.maximum(x.amax(1), -x.amin(1)).float()
    scale = torch.maximum(top / 127, torch.full_like(top, 2.0 ** -126))
    v = x.to(torch.float64) / scale.to(torch.float64).unsqueeze(1)
    low = torch.floor(v)
    up = (v - low > 0.5) | ((v - low == 0.5) & (low % 2 != 0))
    return torch.clip(low + up, -127, 127), scale


def exact(case, seed):
    c = dict(BASE, **case)
    s = _inputs(c, seed)
    f64 = torch.float64
    if c["op"] == "norm":
        return _exact_norm(c, s)
    if c["op"] == "quantize":
        q, scale = [], []
        for lo in range(0, c["rows"], 16384):
            a, b = _exact_quantized(s["x"][lo:lo + 16384])
            q.append(a.to(torch.int8))
            scale.append(b)
        return {"q": torch.cat(q), "scale": torch.cat(scale)}
    if c["op"] == "int8":
        q, scale = (s["x"], s["x_scale"]) if c["given"] else _exact_quantized(s["x"])
        left = q.to(f64) * scale.to(f64)[:, None]
        right = s["weight"].to(f64) * s["weight_scale"].to(f64)[:, None]
        bias = torch.zeros(c["outer"], dtype=f64, device=DEVICE) if s["bias"] is None else s["bias"]
        z = torch.addmm(bias.to(f64), left, right.t().contiguous())
        y = _exact_act(c["activation"], z)
        return {"out": y if s["residual"] is None else s["residual"].to(f64) + y}
    # The polynomial on the eigenvalues of the smaller Gram matrix would divide by small ones;
    # the iteration itself in 64 bits, by Horner's rule on the side that is smaller.
    if c["batch"] * c["steps"] * 6.0 * min(c["rows"], c["inner"]) * c["rows"] * c["inner"] > 6e12:
        return {"out": None}
    p1, p3, p5 = COEFFICIENTS
    out = []
    for i in range(c["batch"]):
        x = s["x"][i].to(f64)
        x = x / (torch.linalg.vector_norm(x) + TINY)
        wide = x.shape[0] <= x.shape[1]
        one = torch.eye(min(x.shape), dtype=f64, device=DEVICE)
        for _ in range(c["steps"]):
            gram = x @ x.t().contiguous() if wide else x.t().contiguous() @ x
            poly = p1 * one + gram @ (p3 * one + p5 * gram)
            x = poly @ x if wide else x @ poly
        out.append(x if s["base"] is None else torch.lerp(-2.0 * x, s["base"][i].to(f64), 0.99))
    return {"out": torch.stack(out)}
