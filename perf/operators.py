"""Measured cases of the layer operators: layer norm, gated feed-forward block, dropout.

Rows are nodes or tokens and features are contiguous, as in the dense operands of the sparse
product. Sizes are this repository's own: the graph's 2^20 nodes with 128 features, the pruned
language model's 4096 x 11008 weight with 1 to 2048 tokens, and ragged ones between.

`run` computes each operator in its plain form (elementary torch operations in 32 bits, rounded
once at the end); with `own` set it calls the framework. `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-5
_M32 = 0xFFFFFFFF
_ACTS = ("silu", "gelu", "relu", "sigmoid")


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # one token's hidden state in front of a feed-forward block: launch latency
        {"name": "norm-token", "op": "norm", "rows": 1, "cols": 4096, "x": "bf16", "y": "bf16"},
        # the graph's aggregated features (fp32, as the sparse product leaves them) normalised
        # into the 16-bit operand of the next product
        {"name": "norm-graph", "op": "norm", "rows": 1 << 20, "cols": 128, "x": "f32", "y": "f16"},
        # gradient of the norm over a training batch of tokens
        {"name": "norm-grad-tokens", "op": "norm_grad", "rows": 4096, "cols": 4096, "x": "bf16",
         "y": "bf16"},
        # dropout and residual at the end of a graph layer
        {"name": "dropout-graph", "op": "drop", "n": 1 << 27, "t": "f16", "p": 0.1,
         "residual": True},
        # gradient of dropout over a short ragged batch, fp32
        {"name": "dropout-grad-odd", "op": "drop", "n": 37 * 1021, "t": "f32", "p": 0.25,
         "residual": False},
        # gate and up projection of a single decoded token: bound by the weights' bytes
        {"name": "ffn-token", "op": "ffn", "rows": 1, "cols": 4096, "inner": 11008, "t": "f16",
         "act": "silu", "saved": False},
        # the same for a decode batch
        {"name": "ffn-batch", "op": "ffn", "rows": 64, "cols": 4096, "inner": 11008, "t": "bf16",
         "act": "silu", "saved": False},
        # odd widths, as a pruned model's removed channels leave them
        {"name": "ffn-ragged", "op": "ffn", "rows": 301, "cols": 1021, "inner": 2731, "t": "bf16",
         "act": "gelu", "saved": False},
        # forward pass of a training batch, projections kept for the backward pass
        {"name": "ffn-train", "op": "ffn", "rows": 2048, "cols": 4096, "inner": 11008, "t": "bf16",
         "act": "silu", "saved": True},
        # gated layer over every node of the graph, in training
        {"name": "ffn-graph", "op": "ffn", "rows": 1 << 20, "cols": 128, "inner": 128, "t": "f16",
         "act": "silu", "saved": True},
        # backward pass of a training batch of ragged length
        {"name": "ffn-grad-train", "op": "ffn_grad", "rows": 1021, "cols": 4096, "inner": 11008,
         "t": "bf16", "act": "silu"},
        # backward pass of the gated layer over the graph's nodes
        {"name": "ffn-grad-graph", "op": "ffn_grad", "rows": 1 << 20, "cols": 128, "inner": 128,
         "t": "f16", "act": "silu"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "norm_grad", "drop", "ffn", "ffn", "ffn_grad"))
    if op == "drop":
        return {"op": op, "n": _spread(rng, 1000, 1 << 27), "t": rng.choice(("f16", "bf16", "f32")),
                "p": rng.choice((0.0, 0.05, 0.1, 0.25, 0.5)), "residual": rng.random() < 0.6}
    if op in ("norm", "norm_grad"):
        cols = _spread(rng, 16, 16384)
        x = rng.choice(("f16", "bf16", "f32"))
        y = rng.choice(("f16", "bf16", "f32")) if x == "f32" else x
        return {"op": op, "rows": _spread(rng, 1, min(1 << 20, (1 << 27) // cols)), "cols": cols,
                "x": x, "y": y}
    cols, inner = _spread(rng, 32, 4096), _spread(rng, 32, 11008)
    if rng.random() < 0.6:  # widths of most models; the others stay odd or ragged
        cols, inner = -(-cols // 32) * 32, -(-inner // 32) * 32
    most = 92_000_000_000 if op == "ffn" else 46_000_000_000  # multiply-adds of a projection
    most = min(1 << 20, (1 << 27) // max(cols, inner), most // (cols * inner))
    case = {"op": op, "rows": _spread(rng, 1, max(1, most)), "cols": cols, "inner": inner,
            "t": rng.choice(("f16", "bf16")), "act": rng.choice(_ACTS)}
    if op == "ffn":
        case["saved"] = rng.random() < 0.5
    return case


# ---- inputs -----------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    op = case["op"]
    s = {"case": case}
    if op == "drop":
        t = _DT[case["t"]]
        s["x"] = normal(case["n"]).to(t)
        s["residual"] = normal(case["n"]).to(t) if case["residual"] else None
        s["seed"] = seed * 0x9E3779B97F4A7C15 & (1 << 64) - 1
        s["offset"] = seed * 977 + 5
        s["out"] = torch.empty_like(s["x"])
        return s
    rows, cols = case["rows"], case["cols"]
    if op in ("norm", "norm_grad"):
        x = normal(rows, cols)
        x *= 1.5
        x += 0.25 + 0.5 * normal(rows, 1)
        s["x"] = x.to(_DT[case["x"]])
        s["w"] = 1.0 + 0.2 * normal(cols)
        s["b"] = 0.1 * normal(cols)
        s["mean"] = torch.empty(rows, device="cuda")
        s["rstd"] = torch.empty(rows, device="cuda")
        s["out"] = torch.empty(rows, cols, dtype=_DT[case["y"]], device="cuda")
        if op == "norm_grad":
            x = s["x"].float()
            s["mean"] = x.sum(1) / cols
            x = x - s["mean"][:, None]
            s["rstd"] = 1.0 / torch.sqrt((x * x).sum(1) / cols + _EPS)
            s["dy"] = normal(rows, cols).to(_DT[case["y"]])
            s["dw"], s["db"] = torch.empty_like(s["w"]), torch.empty_like(s["b"])
        return s
    t, inner = _DT[case["t"]], case["inner"]
    s["x"] = normal(rows, cols).to(t)
    s["wg"] = (normal(inner, cols) / math.sqrt(cols)).to(t)
    s["wu"] = (normal(inner, cols) / math.sqrt(cols)).to(t)
    s["out"] = torch.empty(rows, inner, dtype=t, device="cuda")
    if op == "ffn":
        kept = case["saved"]
        s["g"] = torch.empty_like(s["out"]) if kept else None
        s["u"] = torch.empty_like(s["out"]) if kept else None
    else:
        s["g"] = s["x"] @ s["wg"].t()
        s["u"] = s["x"] @ s["wu"].t()
        s["dy"] = normal(rows, inner).to(t)
        s["out"] = torch.empty_like(s["x"])
        s["dwg"], s["dwu"] = torch.empty_like(s["wg"]), torch.empty_like(s["wu"])
    return s


# ---- the plain forms ----------------------------------------------------------------------------

def _mul32(a, b):
    """High and low 32 bits of a * b for a constant a and words b, both below 2^32."""
    p, q = b * (a & 0xFFFF), b * (a >> 16)
    return (q + (p >> 16)) >> 16, (p + (q << 16)) & _M32


def _words(n, seed, offset):
    """Words 0..n-1 of Philox4x32-10 (Salmon et al., 2011): word i is word i mod 4 of the block
    whose counter is offset + i // 4 and whose key is seed."""
    c0 = torch.arange((n + 3) // 4, device="cuda", dtype=torch.int64) + offset
    c0, c1 = c0 & _M32, (c0 >> 32) & _M32
    c2 = torch.zeros_like(c0)
    c3 = c2
    k0, k1 = seed & _M32, seed >> 32
    for _ in range(10):
        h0, l0 = _mul32(0xD2511F53, c0)
        h1, l1 = _mul32(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _act(name, v):
    if name == "silu":
        return v * _sigmoid(v)
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return torch.where(v > 0, v, torch.zeros_like(v)) if name == "relu" else _sigmoid(v)


def _act_grad(name, v):
    if name == "silu":
        sg = _sigmoid(v)
        return sg * (1.0 + v * (1.0 - sg))
    if name == "gelu":
        return (0.5 * (1.0 + torch.erf(v * math.sqrt(0.5)))
                + v * torch.exp(-0.5 * v * v) / math.sqrt(2.0 * math.pi))
    if name == "relu":
        return (v > 0).to(v.dtype)
    sg = _sigmoid(v)
    return sg * (1.0 - sg)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "drop":
        p = case["p"]
        keep = _words(case["n"], s["seed"], s["offset"]) >= round(p * 2.0 ** 32)
        y = torch.where(keep, s["x"].float() * (1.0 / (1.0 - p)), 0.0)
        if s["residual"] is not None:
            y = s["residual"].float() + y
        return y.to(s["x"].dtype)
    if op == "norm":
        x = s["x"].float()
        mean = x.sum(1) / case["cols"]
        x = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((x * x).sum(1) / case["cols"] + _EPS)
        return (x * rstd[:, None] * s["w"] + s["b"]).to(_DT[case["y"]]), mean, rstd
    if op == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xh = (s["x"].float() - s["mean"][:, None]) * rstd
        t = dy * s["w"]
        c1, c2 = t.sum(1, keepdim=True) / case["cols"], (t * xh).sum(1, keepdim=True) / case["cols"]
        return (rstd * (t - c1 - xh * c2)).to(s["dy"].dtype), (dy * xh).sum(0), dy.sum(0)
    t, act = s["x"].dtype, case["act"]
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    if op == "ffn":
        g, u = x @ wg.t(), x @ wu.t()
        y = (_act(act, g) * u).to(t)
        return (y, g.to(t), u.to(t)) if case["saved"] else y
    g, u, dy = s["g"].float(), s["u"].float(), s["dy"].float()
    du = dy * _act(act, g)
    dg = dy * u * _act_grad(act, g)
    return (dg @ wg + du @ wu).to(t), (dg.t() @ x).to(t), (du.t() @ x).to(t)


# ---- the framework's calls ------------------------------------------------------------------------

_kept = []


def _framework():
    """The package and the executor that a program keeps."""
    if not _kept:
        import xspmm_b200 as xs
        _kept.extend((xs, xs.CudaExecutor(torch.cuda.current_device())))
    return _kept


def _own(s):
    case = s["case"]
    op = case["op"]
    xs, ex = _framework()
    if op == "drop":
        if s["residual"] is None:
            xs.dropout_backward(ex, s["x"], case["p"], s["seed"], s["offset"], s["out"])
        else:
            xs.dropout(ex, s["x"], case["p"], s["seed"], s["offset"], s["out"],
                       residual=s["residual"])
        return s["out"]
    if op == "norm":
        xs.layer_norm(ex, s["x"], s["w"], s["b"], _EPS, s["out"], mean=s["mean"], rstd=s["rstd"])
        return s["out"], s["mean"], s["rstd"]
    if op == "norm_grad":
        xs.layer_norm_backward(ex, s["dy"], s["x"], s["w"], s["mean"], s["rstd"], s["out"],
                               s["dw"], s["db"])
        return s["out"], s["dw"], s["db"]
    if op == "ffn":
        xs.gated_ffn(ex, s["x"], s["wg"], s["wu"], s["out"], activation=case["act"], gate=s["g"],
                     up=s["u"])
        return (s["out"], s["g"], s["u"]) if case["saved"] else s["out"]
    xs.gated_ffn_backward(ex, s["dy"], s["x"], s["wg"], s["wu"], s["g"], s["u"], s["out"],
                          s["dwg"], s["dwu"], activation=case["act"])
    return s["out"], s["dwg"], s["dwu"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "drop":
        size = _BYTES[case["t"]]
        return {"bytes": case["n"] * size * (3 if case["residual"] else 2), "flops": 2 * case["n"]}
    r, c = case["rows"], case["cols"]
    if op in ("norm", "norm_grad"):
        sx, sy = _BYTES[case["x"]], _BYTES[case["y"]]
        if op == "norm":
            return {"bytes": r * c * (sx + sy) + 8 * (r + c), "flops": 8 * r * c}
        return {"bytes": r * c * (sx + 2 * sy) + 8 * r + 12 * c, "flops": 15 * r * c}
    f = case["inner"]
    if op == "ffn":
        outs = 3 if case["saved"] else 1
        return {"bytes": 2 * (r * c + 2 * f * c + outs * r * f), "flops": 4 * r * c * f}
    return {"bytes": 2 * (3 * r * f + 2 * r * c + 4 * f * c), "flops": 8 * r * c * f}


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def _exact_words(n, seed, offset):
    """The same generator with the products taken limb by limb, 2^22 blocks at a time."""
    def product(m, v):
        ml, mh, vl, vh = m % 65536, m // 65536, v % 65536, v // 65536
        low, mid1, mid2, high = ml * vl, ml * vh, mh * vl, mh * vh
        carry = low // 65536 + mid1 % 65536 + mid2 % 65536
        return (high + mid1 // 65536 + mid2 // 65536 + carry // 65536,
                (carry % 65536) * 65536 + low % 65536)

    total, parts = -(-n // 4), []
    for first in range(0, total, 1 << 22):
        at = torch.arange(first, min(total, first + (1 << 22)), device="cuda") + offset
        word = [at % 2 ** 32, at // 2 ** 32, torch.zeros_like(at), torch.zeros_like(at)]
        for r in range(10):
            ka = (seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32
            kb = (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32
            ha, la = product(0xD2511F53, word[0])
            hb, lb = product(0xCD9E8D57, word[2])
            word = [hb ^ word[1] ^ ka, lb, ha ^ word[3] ^ kb, la]
        parts.append(torch.stack(word, dim=-1).flatten())
    return torch.cat(parts)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = {k: v.double() for k, v in s.items()
         if isinstance(v, torch.Tensor) and k in ("x", "w", "b", "dy", "wg", "wu", "g", "u", "residual")
         and not (op == "ffn" and k in ("g", "u"))}
    if op == "drop":
        kept = (_exact_words(case["n"], s["seed"], s["offset"]).double()
                >= float(round(case["p"] * 4294967296))).double()
        y = kept * d["x"] / (1.0 - case["p"])
        return y + d["residual"] if "residual" in d else y
    if op == "norm":
        mean = d["x"].mean(dim=1)
        var = d["x"].var(dim=1, unbiased=False)
        rstd = (var + _EPS).rsqrt()
        return (d["x"] - mean.unsqueeze(1)) / (var + _EPS).sqrt().unsqueeze(1) * d["w"] + d["b"], \
            mean, rstd
    if op == "norm_grad":
        rstd = s["rstd"].double().unsqueeze(1)
        xh = (d["x"] - s["mean"].double().unsqueeze(1)) * rstd
        t = d["dy"] * d["w"]
        dx = rstd * (t - t.mean(dim=1, keepdim=True) - xh * (t * xh).mean(dim=1, keepdim=True))
        return dx, torch.einsum("rc,rc->c", d["dy"], xh), d["dy"].sum(dim=0)
    act = case["act"]
    value = {"silu": lambda v: v / (1 + (-v).exp()),
             "gelu": lambda v: v * 0.5 * torch.special.erfc(-v / math.sqrt(2)),
             "relu": lambda v: v.clamp(min=0),
             "sigmoid": lambda v: 1 / (1 + (-v).exp())}[act]
    if op == "ffn":
        g, u = torch.einsum("tk,fk->tf", d["x"], d["wg"]), torch.einsum("tk,fk->tf", d["x"], d["wu"])
        y = value(g) * u
        return (y, g, u) if case["saved"] else y
    leaf = d["g"].requires_grad_()
    a = value(leaf)
    (slope,) = torch.autograd.grad(a.sum(), leaf)
    dg, du = d["dy"] * d["u"] * slope, d["dy"] * a.detach()
    return (torch.einsum("tf,fk->tk", dg, d["wg"]) + torch.einsum("tf,fk->tk", du, d["wu"]),
            torch.einsum("tf,tk->fk", dg, d["x"]), torch.einsum("tf,tk->fk", du, d["x"]))
