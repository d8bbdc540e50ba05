"""Measured cases of the layer operators: group norm with an activation, quantisation of rows to 8
bits and the product of 8-bit operands, and the orthogonalised update of a weight matrix.

Rows are nodes or tokens and features are contiguous, as in the dense operands of the sparse
product; a batch of graphs is packed, its graphs' rows one after the other. Sizes are this
repository's own: the graph's 2^20 nodes with 128 features, the language model's 4096 x 11008
weight with 1 to 2048 tokens, and ragged ones between.

`run` computes each operator in its plain form (elementary torch operations); with `own` set it
calls the framework. `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-5          # of the norm's variance
_NORM_EPS = 1e-7     # of the update's norm
_NS = (3.4445, -4.7750, 2.0315)  # the Newton-Schulz polynomial's coefficients
_ACTS = (None, "silu", "gelu", "relu", "sigmoid")


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # the whole graph's aggregated features (fp32, as the sparse product leaves them)
        # normalised and activated into the 16-bit operand of the next product
        {"name": "gnorm-graph", "op": "gnorm", "rows": 1 << 20, "cols": 128, "groups": 32,
         "samples": 1, "skew": 0.0, "slack": 0, "x": "f32", "y": "f16", "act": "silu"},
        # a batch of small graphs of different sizes, packed and padded at its end
        {"name": "gnorm-batch", "op": "gnorm", "rows": 1 << 18, "cols": 256, "groups": 32,
         "samples": 4096, "skew": 0.8, "slack": 1021, "x": "bf16", "y": "bf16", "act": "gelu"},
        # gradient over one small graph with an odd group width: launch latency
        {"name": "gnorm-grad-odd", "op": "gnorm_grad", "rows": 301, "cols": 84, "groups": 12,
         "samples": 1, "skew": 0.0, "slack": 0, "x": "f32", "y": "f32", "act": "silu"},
        # gradient over the batch of graphs
        {"name": "gnorm-grad-batch", "op": "gnorm_grad", "rows": 1 << 18, "cols": 256,
         "groups": 32, "samples": 4096, "skew": 0.8, "slack": 0, "x": "bf16", "y": "bf16",
         "act": "silu"},
        # gradient over the whole graph's nodes
        {"name": "gnorm-grad-graph", "op": "gnorm_grad", "rows": 1 << 20, "cols": 128,
         "groups": 32, "samples": 1, "skew": 0.0, "slack": 0, "x": "f16", "y": "f16",
         "act": "relu"},
        # one token's hidden state in front of an 8-bit projection: launch latency
        {"name": "quant-token", "op": "quant", "rows": 1, "cols": 4096, "x": "bf16"},
        # every node's features
        {"name": "quant-graph", "op": "quant", "rows": 1 << 20, "cols": 128, "x": "f32"},
        # projection of a single decoded token: bound by the weight's bytes
        {"name": "int8-token", "op": "int8", "rows": 1, "cols": 4096, "inner": 11008, "y": "f16",
         "bias": True},
        # odd widths, as a pruned model's removed channels leave them, to fp32
        {"name": "int8-ragged", "op": "int8", "rows": 301, "cols": 1021, "inner": 2731,
         "y": "f32", "bias": True},
        # projection of a batch of prompts
        {"name": "int8-tokens", "op": "int8", "rows": 2048, "cols": 4096, "inner": 11008,
         "y": "bf16", "bias": False},
        # update of a graph layer's square projection
        {"name": "update-graph", "op": "update", "rows": 128, "cols": 128, "x": "bf16",
         "y": "bf16"},
        # update of the language model's weight from its fp32 momentum
        {"name": "update-weight", "op": "update", "rows": 11008, "cols": 4096, "x": "f32",
         "y": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("gnorm", "gnorm", "gnorm_grad", "gnorm_grad", "quant", "int8", "int8",
                     "update", "update"))
    if op in ("gnorm", "gnorm_grad"):
        groups, wide = _spread(rng, 1, 64), _spread(rng, 1, 64)
        if rng.random() < 0.5:  # widths of most models; the others stay odd
            groups, wide = -(-groups // 4) * 4, -(-wide // 4) * 4
        cols = groups * wide
        rows = _spread(rng, 1, min(1 << 20, (1 << 27) // cols))
        x = rng.choice(("f16", "bf16", "f32"))
        y = rng.choice(("f16", "bf16", "f32")) if x == "f32" else x
        return {"op": op, "rows": rows, "cols": cols, "groups": groups,
                "samples": 1 if rng.random() < 0.3 else _spread(rng, 1, rows),
                "skew": rng.choice((0.0, 0.5, 1.0, 2.0)),
                "slack": rng.choice((0, 0, 1, 37)), "x": x, "y": y, "act": rng.choice(_ACTS)}
    if op == "quant":
        cols = _spread(rng, 16, 16384)
        return {"op": op, "rows": _spread(rng, 1, min(1 << 20, (1 << 27) // cols)), "cols": cols,
                "x": rng.choice(("f16", "bf16", "f32"))}
    if op == "int8":
        cols, inner = _spread(rng, 16, 11008), _spread(rng, 16, 11008)
        if rng.random() < 0.6:
            cols, inner = -(-cols // 32) * 32, -(-inner // 32) * 32
        most = min(1 << 20, (1 << 27) // max(cols, inner), 92_000_000_000 // (cols * inner))
        return {"op": op, "rows": _spread(rng, 1, max(1, most)), "cols": cols, "inner": inner,
                "y": rng.choice(("f16", "bf16", "f32")), "bias": rng.random() < 0.5}
    small = _spread(rng, 1, 4096)
    large = _spread(rng, small, 11008)
    if rng.random() < 0.6:
        small, large = -(-small // 16) * 16, -(-large // 16) * 16
    rows, cols = (small, large) if rng.random() < 0.5 else (large, small)
    x = rng.choice(("f16", "bf16", "f32"))
    return {"op": op, "rows": rows, "cols": cols, "x": x,
            "y": rng.choice(("f16", "bf16")) if x == "f32" else x}


# ---- inputs -----------------------------------------------------------------------------------

def _offsets(case, g):
    """Where each packed sample begins, and the end: lengths in log-normal proportions."""
    rows, samples = case["rows"], case["samples"]
    share = torch.exp(case["skew"] * torch.randn(samples, generator=g, device="cuda",
                                                 dtype=torch.float64))
    ends = torch.round(share.cumsum(0) / share.sum() * rows).long()
    ends[-1] = rows
    return torch.cat((torch.zeros_like(ends[:1]), ends))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    op = case["op"]
    s = {"case": case}
    if op == "quant":
        # tokens of different sizes, with a few channels that stand out
        x = normal(case["rows"], case["cols"]) * torch.exp(0.5 * normal(case["rows"], 1))
        x *= 1.0 + 3.0 * (normal(case["cols"]) > 2.0)
        s["x"] = x.to(_DT[case["x"]])
        s["q"] = torch.empty(x.shape, dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(case["rows"], device="cuda")
        return s
    if op == "int8":
        rows, cols, inner = case["rows"], case["cols"], case["inner"]
        s["x"] = (normal(rows, cols) * 32.0).round().clamp(-127, 127).to(torch.int8)
        s["w"] = (normal(inner, cols) * 32.0).round().clamp(-127, 127).to(torch.int8)
        s["xs"] = torch.exp(0.5 * normal(rows)) / 32.0
        s["ws"] = torch.exp(0.2 * normal(inner)) / (32.0 * math.sqrt(cols))
        s["b"] = 0.1 * normal(inner) if case["bias"] else None
        s["out"] = torch.empty(rows, inner, dtype=_DT[case["y"]], device="cuda")
        return s
    if op == "update":
        # a gradient or momentum: a few strong directions over noise
        rows, cols = case["rows"], case["cols"]
        x = normal(rows, cols)
        x += (normal(rows, 4) * 2.0) @ normal(4, cols)
        s["x"] = (x * 1e-3).to(_DT[case["x"]])
        s["out"] = torch.empty(rows, cols, dtype=_DT[case["y"]], device="cuda")
        return s
    rows, cols, groups, samples = (case[k] for k in ("rows", "cols", "groups", "samples"))
    total = rows + case["slack"]
    off = _offsets(case, g)
    x = normal(total, cols)
    x *= 1.5
    x += 0.25 + 0.5 * normal(cols)
    s["x"] = x.to(_DT[case["x"]])
    s["off"] = off
    s["w"] = 1.0 + 0.2 * normal(cols)
    s["b"] = 0.1 * normal(cols)
    # rows behind the last sample are left as they are: zeros
    s["out"] = torch.zeros(total, cols, dtype=_DT[case["y"]], device="cuda")
    s["mean"] = torch.empty(samples, groups, device="cuda")
    s["rstd"] = torch.empty(samples, groups, device="cuda")
    if op == "gnorm_grad":
        s["mean"], s["rstd"] = (v.float() for v in _statistics(s["x"], off, case))
        s["dy"] = normal(total, cols).to(_DT[case["y"]])
        s["dw"], s["db"] = torch.empty_like(s["w"]), torch.empty_like(s["b"])
    return s


# ---- the plain forms ----------------------------------------------------------------------------

def _sample_of_rows(off, rows):
    """The sample each of the first `rows` rows lies in."""
    at = torch.arange(off.numel() - 1, device="cuda")
    return torch.repeat_interleave(at, off[1:] - off[:-1], output_size=rows)


def _sample_sums(v, off):
    """Sums over each sample's rows of v, in 64 bits."""
    v = v.double()
    if off.numel() == 2:
        return v.sum(0, keepdim=True)
    c = v.t().contiguous().cumsum(1).t()
    c = torch.cat((torch.zeros_like(c[:1]), c))
    return c[off[1:]] - c[off[:-1]]


def _group_sums(v, groups):
    return v.view(v.shape[0], groups, -1).sum(2)


def _statistics(x, off, case):
    """Mean and 1 / sqrt(var + eps) of each sample's groups, in 64 bits; 0 and 1 / sqrt(eps) where a
    sample has no rows."""
    rows, cols, groups = case["rows"], case["cols"], case["groups"]
    x = x[:rows].float()
    n = (off[1:] - off[:-1]).clamp(min=1)[:, None].double() * (cols // groups)
    mean = _sample_sums(_group_sums(x, groups), off) / n
    of_row = _sample_of_rows(off, rows)
    d = x.view(rows, groups, -1) - mean.float()[of_row][:, :, None]
    var = _sample_sums((d * d).sum(2), off) / n
    return mean, 1.0 / torch.sqrt(var + _EPS)


def _act(name, v):
    if name is None:
        return v
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return v.clamp(min=0.0) if name == "relu" else 1.0 / (1.0 + torch.exp(-v))


def _act_grad(name, v):
    if name is None:
        return torch.ones_like(v)
    if name == "relu":
        return (v > 0).to(v.dtype)
    if name == "gelu":
        return (0.5 * (1.0 + torch.erf(v * math.sqrt(0.5)))
                + v * torch.exp(-0.5 * v * v) / math.sqrt(2.0 * math.pi))
    s = 1.0 / (1.0 + torch.exp(-v))
    return s * (1.0 + v * (1.0 - s)) if name == "silu" else s * (1.0 - s)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quant":
        x = s["x"].float()
        most = torch.abs(x).amax(1, keepdim=True)
        # whole numbers next to a border: the quotient in 64 bits
        q = torch.round(127.0 * x.double() / most.double().clamp(min=1e-300))
        return q.to(torch.int8), (most / 127.0)[:, 0]
    if op == "int8":
        # sums of whole numbers beyond 2^24
        acc = s["x"].double() @ s["w"].double().t()
        y = acc * s["xs"].double()[:, None] * s["ws"].double()
        if s["b"] is not None:
            y = y + s["b"].double()
        return y.to(s["out"].dtype)
    if op == "update":
        x = s["x"].float()
        tall = x.shape[0] > x.shape[1]
        if tall:
            x = x.t()
        x = x / (torch.sqrt((x.double() * x.double()).sum()) + _NORM_EPS).float()
        for _ in range(5):
            a = x @ x.t()
            x = _NS[0] * x + (_NS[1] * a + _NS[2] * (a @ a)) @ x
        return (x.t() if tall else x).to(s["out"].dtype)
    rows, cols, groups = case["rows"], case["cols"], case["groups"]
    off = s["off"]
    of_row = _sample_of_rows(off, rows)
    out = torch.zeros(s["x"].shape, dtype=s["out"].dtype, device="cuda")
    if op == "gnorm":
        mean, rstd = (v.float() for v in _statistics(s["x"], off, case))
    else:
        mean, rstd = s["mean"], s["rstd"]
    xh = (s["x"][:rows].float().view(rows, groups, -1) - mean[of_row][:, :, None]) \
        * rstd[of_row][:, :, None]
    xh = xh.view(rows, cols)
    z = xh * s["w"] + s["b"]
    if op == "gnorm":
        out[:rows] = _act(case["act"], z).to(out.dtype)
        return out, mean, rstd
    dz = s["dy"][:rows].float() * _act_grad(case["act"], z)
    n = (off[1:] - off[:-1]).clamp(min=1)[:, None].double() * (cols // groups)
    t = dz * s["w"]
    c1 = (_sample_sums(_group_sums(t, groups), off) / n).float()[of_row][:, :, None]
    c2 = (_sample_sums(_group_sums(t * xh, groups), off) / n).float()[of_row][:, :, None]
    dx = rstd[of_row][:, :, None] * (t.view(rows, groups, -1) - c1
                                     - xh.view(rows, groups, -1) * c2)
    out[:rows] = dx.view(rows, cols).to(out.dtype)
    return out, (dz * xh).sum(0), dz.sum(0)


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
    if op == "quant":
        xs.quantize_rows(ex, s["x"], s["q"], s["scale"])
        return s["q"], s["scale"]
    if op == "int8":
        xs.linear_int8(ex, s["x"], s["xs"], s["w"], s["ws"], s["out"], bias=s["b"])
        return s["out"]
    if op == "update":
        xs.orthogonalize(ex, s["x"], s["out"], steps=5, eps=_NORM_EPS)
        return s["out"]
    # one sample that takes every row needs no offsets
    off = None if case["samples"] == 1 and case["slack"] == 0 else s["off"]
    if op == "gnorm":
        xs.group_norm(ex, s["x"], case["groups"], s["w"], s["b"], _EPS, s["out"], offsets=off,
                      activation=case["act"], mean=s["mean"], rstd=s["rstd"])
        return s["out"], s["mean"], s["rstd"]
    xs.group_norm_backward(ex, s["dy"], s["x"], case["groups"], s["w"], s["b"], s["mean"],
                           s["rstd"], s["out"], s["dw"], s["db"], offsets=off,
                           activation=case["act"])
    return s["out"], s["dw"], s["db"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------

def work(case):
    op = case["op"]
    r, c = case["rows"], case["cols"]
    if op == "quant":
        return {"bytes": r * c * (_BYTES[case["x"]] + 1) + 4 * r, "flops": 3 * r * c}
    if op == "int8":
        f = case["inner"]
        return {"bytes": r * c + f * c + r * f * _BYTES[case["y"]] + 4 * (r + 2 * f),
                "flops": 2 * r * c * f}
    if op == "update":
        m, n = min(r, c), max(r, c)
        # a step: half of the symmetric X X^T and of A A, and B X
        return {"bytes": r * c * (_BYTES[case["x"]] + _BYTES[case["y"]]),
                "flops": 5 * (m * (m + 1) * (n + m) + 2 * m * m * n)}
    sx, sy = _BYTES[case["x"]], _BYTES[case["y"]]
    few = 8 * case["samples"] * (case["groups"] + 1)
    if op == "gnorm":
        return {"bytes": r * c * (sx + sy) + 8 * c + few, "flops": 10 * r * c}
    return {"bytes": r * c * (sx + 2 * sy) + 16 * c + few, "flops": 18 * r * c}


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        x = s["x"].double()
        return None, x.abs().max(dim=1).values / 127.0
    if op == "int8":
        y = torch.einsum("rk,fk->rf", s["x"].double() * s["xs"].double().unsqueeze(1),
                         s["w"].double() * s["ws"].double().unsqueeze(1))
        return y if s["b"] is None else y + s["b"].double().unsqueeze(0)
    if op == "update":
        x = s["x"].double()
        x = x / (torch.linalg.matrix_norm(x) + _NORM_EPS)
        a, b, c = _NS
        for _ in range(5):
            if case["rows"] <= case["cols"]:
                gram = torch.einsum("ik,jk->ij", x, x)
                x = a * x + torch.einsum("ij,jk->ik", gram, b * x + c * torch.einsum(
                    "ij,jk->ik", gram, x))
            else:
                gram = torch.einsum("ki,kj->ij", x, x)
                x = a * x + torch.einsum("ki,ij->kj", b * x + c * torch.einsum(
                    "ki,ij->kj", x, gram), gram)
        return x
    rows, cols, groups, samples = (case[k] for k in ("rows", "cols", "groups", "samples"))
    bounds = s["off"]
    where = torch.searchsorted(bounds[1:].contiguous(), torch.arange(rows, device="cuda"), right=True)
    count = torch.zeros(samples, dtype=torch.float64, device="cuda")
    count = count.index_add(0, where, torch.ones(rows, dtype=torch.float64, device="cuda"))
    count = (count * (cols // groups)).clamp(min=1.0).unsqueeze(1)

    def total(v):  # over each sample's rows and the group's columns
        v = v.reshape(rows, groups, cols // groups).sum(dim=-1)
        if samples == 1:
            return v.sum(dim=0, keepdim=True)
        return torch.zeros(samples, groups, dtype=torch.float64, device="cuda").index_add(0, where, v)

    def spread(v):  # a value of each sample and group to its rows and columns
        return v[where].repeat_interleave(cols // groups, dim=1)

    x, w, b = s["x"][:rows].double(), s["w"].double(), s["b"].double()
    value = {None: lambda v: v, "silu": lambda v: v * torch.special.expit(v),
             "gelu": lambda v: v * 0.5 * torch.special.erfc(-v / math.sqrt(2)),
             "relu": lambda v: v.clamp(min=0), "sigmoid": torch.special.expit}[case["act"]]
    out = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    if op == "gnorm":
        mean = total(x) / count
        var = total((x - spread(mean)) ** 2) / count
        z = (x - spread(mean)) / spread((var + _EPS).sqrt()) * w + b
        out[:rows] = value(z)
        return out, mean, (var + _EPS).rsqrt()
    mean, rstd = s["mean"].double(), s["rstd"].double()
    xh = (x - spread(mean)) * spread(rstd)
    leaf = (xh * w + b).requires_grad_()
    (slope,) = torch.autograd.grad(value(leaf).sum(), leaf)
    dz = s["dy"][:rows].double() * slope
    t = dz * w
    dx = t - spread(total(t) / count) - xh * spread(total(t * xh) / count)
    out[:rows] = dx * spread(rstd)
    return out, torch.einsum("rc,rc->c", dz, xh), dz.sum(dim=0)
