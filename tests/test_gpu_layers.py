"""GPU tests of the layer operators (layer norm, dropout, gated feed-forward) against plain
restatements in 64 bits.

Tolerances, element by element. U[T] is the largest relative error of one rounding to type T
(2^-11 fp16, 2^-8 bf16, 2^-24 fp32), TINY[T] the largest absolute one among its subnormals. A sum of n
fp32 terms is within n * 2^-23 of the sum of their magnitudes: 2^-24 for each rounding, doubled because
the tensor core's additions are not specified to round to nearest. E = 2^-20 covers the dozen fp32
roundings and the exponential of an elementwise formula. An output is within its formula's error plus
U[T] of its own magnitude (1.01 covers the products of errors).
"""
import math

import numpy as np
import pytest
import torch

import xspmm_b200 as xs
from xspmm_b200 import _lib

pytestmark = pytest.mark.gpu

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32
U = {f16: 2.0 ** -11, bf16: 2.0 ** -8, f32: 2.0 ** -24}
TINY = {f16: 2.0 ** -25, bf16: 2.0 ** -134, f32: 2.0 ** -150}
E, S = 2.0 ** -20, 2.0 ** -23


def rand(seed, *shape, dtype=f32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def close(got, ref, err, what=""):
    """got (type T) within 1.01 * (err + U[T] * |ref|) of ref (64 bits)."""
    T = got.dtype
    tol = 1.01 * (err + U[T] * ref.abs()) + TINY[T]
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: off by {off.max().item():.3e}, over the bound by {worst:.3e}"


def guarded(rows, cols, dtype, ld=None, fill=7.0):
    """A rows x cols view with row stride ld inside a buffer of `fill`, and the buffer."""
    ld = ld or cols
    buf = torch.full((rows * ld + 64,), fill, dtype=dtype, device="cuda")
    return buf.as_strided((rows, cols), (ld, 1)), buf


def outside_untouched(view, buf, fill=7.0):
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep.as_strided(view.shape, view.stride()).fill_(False)
    assert bool((buf[keep] == fill).all()), "written outside the output"


# ---- layer norm ---------------------------------------------------------------------------------

NORM_TYPES = [(f16, f16), (bf16, bf16), (f32, f32), (f32, f16), (f32, bf16)]
NORM_SIZES = [(1, 1), (1, 4096), (3, 7), (5, 32), (257, 128), (64, 129), (33, 1000), (9, 1021),
              (7, 2048), (1000, 24), (3, 5003), (2, 8193), (3, 16384), (2, 20001), (2, 40000), (1500, 64)]


def norm_ref(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    return mean, rstd, d * rstd * w.double() + b.double()


@pytest.mark.parametrize("tx,ty", NORM_TYPES)
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_layer_norm(executor, rows, cols, tx, ty):
    x = rand(rows * 31 + cols, rows, cols, dtype=tx, scale=1.5, shift=0.25)
    w, b = rand(1, cols, scale=0.2, shift=1.0), rand(2, cols, scale=0.1)
    y, buf = guarded(rows, cols, ty)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    xs.layer_norm(executor, x, w, b, 1e-5, y, mean=mean, rstd=rstd)
    rm, rr, ref = norm_ref(x, w, b, 1e-5)
    mag = x.double().abs().mean(1, keepdim=True)
    em = cols * S * mag + E * rm.abs()
    # rstd: relative error of half the variance's own (a sum of squares of x - mean)
    er = rr * (cols * S + em * rr + E)
    close(mean[:, None], rm, em, "mean")
    close(rstd[:, None], rr, er, "rstd")
    xh = (x.double() - rm) * rr
    close(y, ref, w.double().abs() * (em * rr + xh.abs() * (er / rr) + E * xh.abs()) + E * ref.abs()
          + E * b.double().abs(), "y")
    outside_untouched(y, buf)


@pytest.mark.parametrize("tx,ty", NORM_TYPES)
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_layer_norm_backward(executor, rows, cols, tx, ty):
    x = rand(rows * 37 + cols, rows, cols, dtype=tx, scale=1.5, shift=0.25)
    dy = rand(rows * 41 + cols, rows, cols, dtype=ty)
    w = rand(1, cols, scale=0.2, shift=1.0)
    m64, r64, _ = norm_ref(x, w, w, 1e-5)
    mean, rstd = m64[:, 0].float(), r64[:, 0].float()
    dx, buf = guarded(rows, cols, ty)
    dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    xs.layer_norm_backward(executor, dy, x, w, mean, rstd, dx, dw, db)
    g, r = dy.double(), rstd.double()[:, None]
    xh = (x.double() - mean.double()[:, None]) * r
    t = g * w.double()
    c1, c2 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
    e1 = (cols * S + E) * t.abs().mean(1, keepdim=True)
    e2 = (cols * S + E) * (t * xh).abs().mean(1, keepdim=True)
    # x - mean cancels: its fp32 rounding is relative to the result (Sterbenz or one rounding)
    close(dx, r * (t - c1 - xh * c2), r * (e1 + xh.abs() * e2 + E * (t.abs() + c1.abs() + (xh * c2).abs())),
          "dx")
    close(dw, (g * xh).sum(0), (rows * S + E) * (g * xh).abs().sum(0), "dweight")
    close(db, g.sum(0), (rows * S + E) * g.abs().sum(0), "dbias")
    outside_untouched(dx, buf)
    # the parts alone are the same numbers
    dw2, dx2 = torch.empty_like(dw), torch.empty_like(dx)
    xs.layer_norm_backward(executor, dy, x, w, mean, rstd, None, dw2, None)
    xs.layer_norm_backward(executor, dy, x, w, mean, rstd, dx2)
    assert torch.equal(dw, dw2) and torch.equal(dx, dx2)


@pytest.mark.parametrize("tx,ty", NORM_TYPES)
@pytest.mark.parametrize("pad", [3, 8])
def test_layer_norm_row_strides(executor, tx, ty, pad):
    """Slices of columns of wider tensors, at aligned and unaligned starts, give the same numbers as
    contiguous copies within the tolerance of y's type, and nothing outside is written."""
    rows, cols = 37, 136
    wide = rand(5, rows, cols + 3 * pad, dtype=tx)
    x = wide[:, pad:pad + cols]
    w, b = rand(1, cols), rand(2, cols)
    y, buf = guarded(rows, cols, ty, ld=cols + pad)
    xs.layer_norm(executor, x, w, b, 1e-5, y)
    dense = torch.empty(rows, cols, dtype=ty, device="cuda")
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    xs.layer_norm(executor, x.contiguous(), w, b, 1e-5, dense, mean, rstd)
    close(y, dense.double(), 2 * cols * S * (1 + dense.double().abs()) + U[ty] * dense.double().abs())
    outside_untouched(y, buf)
    dwide = rand(6, rows, cols + pad, dtype=ty)
    dx, buf = guarded(rows, cols, ty, ld=cols + 2 * pad)
    dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    xs.layer_norm_backward(executor, dwide[:, :cols], x, w, mean, rstd, dx, dw, db)
    ddx, ddw, ddb = torch.empty_like(dense), torch.empty_like(dw), torch.empty_like(db)
    xs.layer_norm_backward(executor, dwide[:, :cols].contiguous(), x.contiguous(), w, mean, rstd, ddx,
                           ddw, ddb)
    close(dx, ddx.double(), 2 * cols * S * 8 + U[ty] * ddx.double().abs())
    close(dw, ddw.double(), 4 * rows * S * rows * torch.ones_like(ddw).double())
    close(db, ddb.double(), 4 * rows * S * rows * torch.ones_like(ddb).double())
    outside_untouched(dx, buf)


@pytest.mark.parametrize("tx,ty", NORM_TYPES)
@pytest.mark.parametrize("rows,cols", [(3001, 2051), (700, 4821), (601, 8191), (5, 16376), (4, 16383)])
def test_layer_norm_long_odd_rows(executor, rows, cols, tx, ty):
    """Rows that start off every boundary, more of them than fit the GPU at once."""
    test_layer_norm(executor, rows, cols, tx, ty)
    test_layer_norm_backward(executor, rows, cols, tx, ty)


def test_layer_norm_without_parameters_in_place_and_empty(executor):
    x = rand(3, 50, 96, dtype=bf16)
    one, zero = torch.ones(96, device="cuda"), torch.zeros(96, device="cuda")
    y1, y2 = torch.empty_like(x), x.clone()
    xs.layer_norm(executor, x, one, zero, 1e-5, y1)
    xs.layer_norm(executor, y2, None, None, 1e-5, y2)
    assert torch.equal(y1, y2)
    mean, rstd = torch.empty(50, device="cuda"), torch.empty(50, device="cuda")
    xs.layer_norm(executor, x, None, None, 1e-5, y1, mean, rstd)
    dy = rand(4, 50, 96, dtype=bf16)
    d1 = torch.empty_like(x)
    xs.layer_norm_backward(executor, dy, x, one, mean, rstd, d1)
    xs.layer_norm_backward(executor, dy, x, None, mean, rstd, dy)
    assert torch.equal(d1, dy)
    dw, db = one.clone(), one.clone()
    none = x[:0]
    xs.layer_norm(executor, none, one, zero, 1e-5, y1[:0])
    xs.layer_norm_backward(executor, none, none, one, mean[:0], rstd[:0], None, dw, db)
    assert not dw.any() and not db.any()


def test_layer_norm_constant_rows_and_not_a_number(executor):
    """A constant row has variance 0 (y = bias); a row with a NaN or Inf does not touch its
    neighbours."""
    x = rand(7, 6, 200, dtype=f16)
    x[1] = 3.0
    x[3, 17] = float("nan")
    x[4, 18] = float("inf")
    w, b = rand(1, 200), rand(2, 200)
    y = torch.empty_like(x)
    mean, rstd = torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    xs.layer_norm(executor, x, w, b, 1e-5, y, mean, rstd)
    assert torch.equal(y[1], b.half())
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).any()
    assert torch.isfinite(y[[0, 1, 2, 5]]).all()
    assert mean[1].item() == 3.0


def test_layer_norm_gradient_against_differences(executor):
    """The directional derivative of sum(dy * y), by central differences of the 64-bit formula."""
    rows, cols, h = 11, 77, 1e-4
    x, dy = rand(1, rows, cols), rand(2, rows, cols)
    w, b = rand(3, cols, shift=1.0, scale=0.3), rand(4, cols)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    xs.layer_norm(executor, x, w, b, 1e-5, y, mean, rstd)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    xs.layer_norm_backward(executor, dy, x, w, mean, rstd, dx, dw, db)
    for at, grad, seed in ((0, dx, 5), (1, dw, 6), (2, db, 7)):
        v = rand(seed, *grad.shape).double()

        def loss(s):
            args = [x.double(), w.double(), b.double()]
            args[at] = args[at] + s * v
            return (dy.double() * norm_ref(*args, 1e-5)[2]).sum()

        num = ((loss(h) - loss(-h)) / (2 * h)).item()
        got = (grad.double() * v).sum().item()
        # fp32 rounding of the gradient and the second-order term of the difference
        assert abs(num - got) <= (grad.double() * v).abs().sum().item() * (rows * cols * S + 10 * h * h) + 1e-6


# ---- dropout ------------------------------------------------------------------------------------

def philox(counters, seed):
    """Philox4x32-10 in numpy, 64-bit counters (uint64) to four words each."""
    m = np.uint64(0xFFFFFFFF)
    c = [counters & m, counters >> np.uint64(32), np.zeros_like(counters), np.zeros_like(counters)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & m,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(-1)


def keep_mask(n, p, seed, offset):
    first = np.uint64(offset) + np.arange((n + 3) // 4, dtype=np.uint64)
    return torch.from_numpy(philox(first, seed)[:n].astype(np.int64) >= round(p * 2 ** 32)).cuda()


def test_philox_known_answers():
    """The generator's published test vectors, for a zero counter and key and for all ones in the
    64 counter bits in use (the latter by a second evaluation in Python integers)."""
    assert [hex(w) for w in philox(np.zeros(1, np.uint64), 0)] == [
        "0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    c, k = [0xFFFFFFFF, 0xFFFFFFFF, 0, 0], [0xFFFFFFFF, 0xFFFFFFFF]
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 % 2 ** 32, (p0 >> 32) ^ c[3] ^ k[1], p0 % 2 ** 32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    assert list(philox(np.full(1, 2 ** 64 - 1, np.uint64), 2 ** 64 - 1)) == c


@pytest.mark.parametrize("dtype", [f16, bf16, f32])
@pytest.mark.parametrize("n", [1, 3, 4, 5, 31, 1000, 4096, 37777, 1 << 20])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(executor, dtype, n, p):
    seed, offset = 0x123456789ABCDEF1 + n, 2 ** 32 - 3  # the counter's high word changes inside
    x, res = rand(n, n, dtype=dtype), rand(n + 1, n, dtype=dtype)
    keep = keep_mask(n, p, seed, offset)
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=f32, device="cuda")
    kept = torch.where(keep, x.float() * scale, torch.zeros((), device="cuda"))
    y, buf = guarded(1, n, dtype)
    y = y[0]
    xs.dropout(executor, x, p, seed, offset, y)
    assert torch.equal(y, kept.to(dtype))  # one product, one rounding: exact
    outside_untouched(y[None], buf)
    xs.dropout(executor, x, p, seed, offset, y, residual=res)
    ref = res.double() + kept.double()
    close(y, ref, 2 * U[f32] * (res.double().abs() + kept.double().abs()))
    dx = torch.empty_like(x)
    xs.dropout_backward(executor, x, p, seed, offset, dx)
    assert torch.equal(dx, kept.to(dtype))


@pytest.mark.parametrize("dtype", [f16, bf16, f32])
@pytest.mark.parametrize("start", [1, 3, 4])
def test_dropout_unaligned_in_place_and_split(executor, dtype, start):
    """Views that start off a 16-byte boundary, y over x or over the residual, and a tensor taken in
    two calls whose offsets follow each other, all give the numbers of one aligned call."""
    n, seed = 5000, 99
    x, res = rand(1, n, dtype=dtype), rand(2, n, dtype=dtype)
    whole = torch.empty_like(x)
    xs.dropout(executor, x, 0.3, seed, 7, whole, residual=res)

    def view(src):
        v = torch.empty(n + 8, dtype=dtype, device="cuda")[start:start + n]
        v.copy_(src)
        return v

    a, r = view(x), view(res)
    xs.dropout(executor, a, 0.3, seed, 7, a, residual=r)
    assert torch.equal(a, whole)
    xs.dropout(executor, view(x), 0.3, seed, 7, r, residual=r)
    assert torch.equal(r, whole)
    parts = torch.empty_like(x)
    xs.dropout(executor, x[:2000], 0.3, seed, 7, parts[:2000], residual=res[:2000])
    xs.dropout(executor, x[2000:], 0.3, seed, 7 + 500, parts[2000:], residual=res[2000:])
    assert torch.equal(parts, whole)
    wrap = torch.empty_like(x)  # counters that pass 2^64 start again at 0
    xs.dropout(executor, x, 0.3, seed, 2 ** 64 - 2, wrap)
    tail = torch.empty_like(x[8:])
    xs.dropout(executor, x[8:], 0.3, seed, 0, tail)
    assert torch.equal(wrap[8:], tail)


def test_dropout_of_infinities_and_nothing(executor):
    x = torch.full((4096,), float("inf"), device="cuda")
    x[::2] = float("nan")
    y = torch.empty_like(x)
    xs.dropout(executor, x, 0.5, 5, 0, y)
    keep = keep_mask(4096, 0.5, 5, 0)
    assert bool((y[~keep] == 0).all()) and not torch.isfinite(y[keep]).any()
    xs.dropout(executor, x[:0], 0.5, 5, 0, y[:0])


# ---- gated feed-forward -------------------------------------------------------------------------

ACTS = {"silu": (lambda v: v * torch.sigmoid(v),
                 lambda v: torch.sigmoid(v) * (1 + v * (1 - torch.sigmoid(v)))),
        "gelu": (lambda v: 0.5 * v * (1 + torch.erf(v / math.sqrt(2))),
                 lambda v: 0.5 * (1 + torch.erf(v / math.sqrt(2)))
                 + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)),
        "relu": (lambda v: v.clamp(min=0), lambda v: (v > 0).double()),
        "sigmoid": (torch.sigmoid, lambda v: torch.sigmoid(v) * (1 - torch.sigmoid(v)))}
FFN_SIZES = [(1, 1, 1), (1, 64, 128), (2, 8, 8), (3, 7, 5), (1, 4096, 11008 // 8), (5, 129, 257),
             (16, 256, 96), (17, 512, 1000), (64, 1000, 264), (65, 96, 128), (100, 72, 40), (127, 128, 128),
             (128, 128, 128), (129, 128, 136), (300, 1021, 517), (1000, 128, 128), (257, 64, 1032),
             (2500, 192, 64), (40, 2048, 2048)]


def ffn_problem(rows, K, F, dtype, seed=0):
    x = rand(seed + rows * 7 + K, rows, K, dtype=dtype)
    wg = rand(seed + F, F, K, dtype=dtype, scale=1.5 / math.sqrt(K))
    wu = rand(seed + F + 1, F, K, dtype=dtype, scale=1.5 / math.sqrt(K))
    return x, wg, wu


def ffn_errors(x, wg, wu, act):
    """64-bit projections and output, and the bound on each one's error before its rounding."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    K = x.shape[1]
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = ((K * S) * (x.abs() @ w.abs().t()) for w in (wg, wu))
    a = ACTS[act][0](g)
    # |act'| <= 1.13 for all four; E relative to |g| + 1 covers the exponential and erf
    ea = 1.13 * eg + E * (g.abs() + 1 if act != "relu" else g.abs())
    return g, u, a * u, eg, eu, ea * u.abs() + (a.abs() + ea) * eu + E * (a * u).abs()


@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("rows,K,F", FFN_SIZES)
def test_gated_ffn(executor, rows, K, F, act, dtype):
    x, wg, wu = ffn_problem(rows, K, F, dtype)
    g, u, ref, eg, eu, ey = ffn_errors(x, wg, wu, act)
    y, buf = guarded(rows, F, dtype)
    xs.gated_ffn(executor, x, wg, wu, y, act)
    close(y, ref, ey, "y")
    outside_untouched(y, buf)
    y2, gate, up = torch.empty_like(y), torch.empty_like(y), torch.empty_like(y)
    xs.gated_ffn(executor, x, wg, wu, y2, act, gate, up)
    close(y2, ref, ey, "y with the projections kept")
    close(gate, g, eg, "gate")
    close(up, u, eu, "up")


def grad_ref(x, wg, wu, gate, up, dy, act, dtype):
    """64-bit gradients and their error bounds. dg and du are rounded to dtype before the products
    and may lie among fp16's subnormals, so each carries U of itself plus TINY."""
    x, wg, wu, g, u, d = (v.double() for v in (x, wg, wu, gate, up, dy))
    rows, F = g.shape
    a, s = ACTS[act][0](g), ACTS[act][1](g)
    dg, du = d * u * s, d * a
    edg = U[dtype] * dg.abs() + 4 * E * (d * u).abs() * (1 + g.abs()) + TINY[dtype]
    edu = U[dtype] * du.abs() + E * d.abs() * (1 + g.abs()) + TINY[dtype]
    dx = dg @ wg + du @ wu
    edx = (edg + 2 * F * S * dg.abs()) @ wg.abs() + (edu + 2 * F * S * du.abs()) @ wu.abs()
    dwg, dwu = dg.t() @ x, du.t() @ x
    edwg = (edg + rows * S * dg.abs()).t() @ x.abs()
    edwu = (edu + rows * S * du.abs()).t() @ x.abs()
    return (dx, edx), (dwg, edwg), (dwu, edwu)


@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("rows,K,F", FFN_SIZES)
def test_gated_ffn_backward(executor, rows, K, F, act, dtype):
    x, wg, wu = ffn_problem(rows, K, F, dtype, seed=50)
    gate, up = (x.float() @ wg.float().t()).to(dtype), (x.float() @ wu.float().t()).to(dtype)
    dy = rand(3, rows, F, dtype=dtype)
    dx, buf = guarded(rows, K, dtype)
    dwg, bg = guarded(F, K, dtype)
    dwu, bu = guarded(F, K, dtype)
    xs.gated_ffn_backward(executor, dy, x, wg, wu, gate, up, dx, dwg, dwu, activation=act)
    for got, (ref, err), name in zip((dx, dwg, dwu), grad_ref(x, wg, wu, gate, up, dy, act, dtype),
                                     ("dx", "dw_gate", "dw_up")):
        close(got, ref, err, name)
    for view, b in ((dx, buf), (dwg, bg), (dwu, bu)):
        outside_untouched(view, b)


@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("rows,K,F", [(1100, 520, 3000), (40003, 128, 120), (30000, 64, 128), (150, 4096, 300)])
def test_gated_ffn_several_waves(executor, rows, K, F, dtype):
    """More tiles than the GPU takes at once, split sums, and several tiles a CTA in the one-pass gradient."""
    test_gated_ffn(executor, rows, K, F, "silu", dtype)
    test_gated_ffn_backward(executor, rows, K, F, "silu", dtype)


@pytest.mark.parametrize("start,pad", [(0, 0), (1, 0), (2, 4), (0, 3), (8, 8)])
@pytest.mark.parametrize("rows,K,F", [(130, 126, 70), (333, 134, 126), (201, 64, 133), (77, 250, 191)])
def test_gated_ffn_odd_widths_and_addresses(executor, rows, K, F, start, pad):
    """Outputs that start at any element with any row stride, beside kept projections, dy and weights'
    gradients at odd addresses: every width a store can have, up to the matrix's last element."""
    def placed(r, c, gap=0):
        buf = torch.full((start + r * (c + gap) + 64,), 7.0, dtype=f16, device="cuda")
        return buf.as_strided((r, c), (c + gap, 1), start), buf

    x, wg, wu = ffn_problem(rows, K, F, f16, seed=9)
    g, u, ref, eg, eu, ey = ffn_errors(x, wg, wu, "silu")
    (y, b0), (gate, b1), (up, b2) = placed(rows, F, pad), placed(rows, F), placed(rows, F)
    xs.gated_ffn(executor, x, wg, wu, y, "silu", gate, up)
    for got, r, e, name in ((y, ref, ey, "y"), (gate, g, eg, "gate"), (up, u, eu, "up")):
        close(got, r, e, name)
    (dy, b3), (dx, b4) = placed(rows, F, pad), placed(rows, K, pad)
    dy.copy_(rand(6, rows, F, dtype=f16))
    (dwg, b5), (dwu, b6) = placed(F, K), placed(F, K)
    xs.gated_ffn_backward(executor, dy, x, wg, wu, gate, up, dx, dwg, dwu)
    for got, (r, e), name in zip((dx, dwg, dwu), grad_ref(x, wg, wu, gate, up, dy, "silu", f16),
                                 ("dx", "dw_gate", "dw_up")):
        close(got, r, e, name)
    for view, buf in ((y, b0), (gate, b1), (up, b2), (dx, b4), (dwg, b5), (dwu, b6)):
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep.as_strided(view.shape, view.stride(), start).fill_(False)
        assert bool((buf[keep] == 7.0).all()), "written outside the output"


@pytest.mark.parametrize("rows", [3, 200])
def test_gated_ffn_parts_strides_and_packed_weights(executor, rows):
    """Both weights as halves of one packed tensor with a row stride, x and y as column slices at
    unaligned places; dx alone and the weights' gradients alone equal the joint call's."""
    K, F = 136, 152
    pack = rand(1, 2 * F, K + 5, dtype=bf16, scale=0.1)
    wg, wu = pack[:F, 1:K + 1], pack[F:, 1:K + 1]
    x = rand(2, rows, K + 9, dtype=bf16)[:, 3:3 + K]
    y, buf = guarded(rows, F, bf16, ld=F + 3)
    xs.gated_ffn(executor, x, wg, wu, y)
    _, _, ref, _, _, ey = ffn_errors(x, wg, wu, "silu")
    close(y, ref, ey)
    outside_untouched(y, buf)
    gate, up = (x.float() @ wg.float().t()).bfloat16(), (x.float() @ wu.float().t()).bfloat16()
    dy = rand(4, rows, F + 7, dtype=bf16)[:, 2:2 + F]
    dx, buf = guarded(rows, K, bf16, ld=K + 1)
    xs.gated_ffn_backward(executor, dy, x, wg, wu, gate, up, dx)
    outside_untouched(dx, buf)
    dwg, dwu = torch.empty(F, K, dtype=bf16, device="cuda"), torch.empty(F, K, dtype=bf16, device="cuda")
    xs.gated_ffn_backward(executor, dy, x, wg, wu, gate, up, None, dwg, dwu)
    for got, (r, e) in zip((dx, dwg, dwu), grad_ref(x, wg, wu, gate, up, dy, "silu", bf16)):
        close(got, r, e)


def test_gated_ffn_of_nothing(executor):
    x, wg, wu = ffn_problem(4, 16, 8, f16)
    y = torch.full((4, 8), 7.0, dtype=f16, device="cuda")
    xs.gated_ffn(executor, x[:0], wg, wu, y[:0])
    xs.gated_ffn(executor, x, wg[:0], wu[:0], y[:, :0])
    assert bool((y == 7).all())
    xs.gated_ffn(executor, x[:, :0], wg[:, :0], wu[:, :0], y)  # sums of no terms
    assert not y.any()
    dwg, dwu = torch.ones_like(wg), torch.ones_like(wu)
    xs.gated_ffn_backward(executor, y[:0], x[:0], wg, wu, y[:0], y[:0], x[:0], dwg, dwu)
    assert not dwg.any() and not dwu.any()
    dx = torch.ones_like(x)
    xs.gated_ffn_backward(executor, y[:, :0], x, wg[:0], wu[:0], y[:, :0], y[:, :0], dx, wg[:0], wu[:0])
    assert not dx.any()


def test_gated_ffn_infinities_stay_in_their_rows(executor):
    """An Inf or NaN in one row of x reaches no other row of y (also where rows share a tile or are
    padding of one)."""
    x, wg, wu = ffn_problem(130, 64, 72, f16)
    y0, y1 = torch.empty(130, 72, dtype=f16, device="cuda"), torch.empty(130, 72, dtype=f16, device="cuda")
    xs.gated_ffn(executor, x, wg, wu, y0)
    x2 = x.clone()
    x2[5, 3] = float("inf")
    x2[129, 60] = float("nan")
    xs.gated_ffn(executor, x2, wg, wu, y1)
    rest = [i for i in range(130) if i not in (5, 129)]
    assert torch.equal(y0[rest], y1[rest])
    assert not torch.isfinite(y1[5]).all() and torch.isnan(y1[129]).all()


def test_gated_ffn_gradient_against_differences(executor):
    rows, K, F, h = 20, 24, 40, 1e-4
    x, wg, wu = ffn_problem(rows, K, F, f16)
    dy = rand(3, rows, F, dtype=f16)
    for act in ACTS:
        gate, up = (x.float() @ wg.float().t()).half(), (x.float() @ wu.float().t()).half()
        dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
        xs.gated_ffn_backward(executor, dy, x, wg, wu, gate, up, dx, dwg, dwu, activation=act)
        bounds = grad_ref(x, wg, wu, gate, up, dy, act, f16)
        # the kept projections are rounded to fp16, which moves the slopes the formula uses
        exact = grad_ref(x, wg, wu, x.double() @ wg.double().t(), x.double() @ wu.double().t(), dy, act, f16)
        for at, grad in enumerate((dx, dwg, dwu)):
            v = rand(60 + at, *grad.shape).double()

            def loss(s):
                args = [x.double(), wg.double(), wu.double()]
                args[at] = args[at] + s * v
                return (dy.double() * ACTS[act][0](args[0] @ args[1].t()) * (args[0] @ args[2].t())).sum()

            num = ((loss(h) - loss(-h)) / (2 * h)).item()
            got = (grad.double() * v).sum().item()
            tol = ((bounds[at][1] + U[f16] * bounds[at][0].abs() + (bounds[at][0] - exact[at][0]).abs())
                   * v.abs()).sum().item()
            kink = 0.0
            if act == "relu":  # terms whose gate changes sign within the step
                g = x.double() @ wg.double().t()
                kink = (dy.double() * (x.double() @ wu.double().t()))[g.abs() < 1e-2].abs().sum().item()
            assert abs(num - got) <= tol + kink + 1e-3 * h / 1e-4, (act, at)


# ---- the manner of the calls --------------------------------------------------------------------

def test_large_offsets(executor):
    """Elements past 2^31 of a matrix with a large row stride are found (64-bit index arithmetic)."""
    ld = (1 << 30) + 8
    buf = torch.zeros(2 * ld + 128, dtype=bf16, device="cuda")
    x = buf.as_strided((3, 64), (ld, 1))
    x.copy_(rand(1, 3, 64, dtype=bf16))
    w = rand(2, 64)
    y, y2 = torch.empty(3, 64, dtype=bf16, device="cuda"), torch.empty(3, 64, dtype=bf16, device="cuda")
    xs.layer_norm(executor, x, w, w, 1e-5, y)
    xs.layer_norm(executor, x.contiguous(), w, w, 1e-5, y2)
    assert torch.equal(y, y2)
    wg, wu = rand(3, 24, 64, dtype=bf16), rand(4, 24, 64, dtype=bf16)
    h, h2 = torch.empty(3, 24, dtype=bf16, device="cuda"), torch.empty(3, 24, dtype=bf16, device="cuda")
    xs.gated_ffn(executor, x, wg, wu, h)
    xs.gated_ffn(executor, x.contiguous(), wg, wu, h2)
    assert torch.equal(h, h2)


def test_runs_on_the_current_stream(executor):
    """The call waits for the work already enqueued on torch's current stream, and counts its
    launches."""
    s = torch.cuda.Stream()
    x, y = torch.zeros(1 << 22, device="cuda"), torch.empty(1 << 22, device="cuda")
    torch.cuda.synchronize()
    before = executor.launch_count()
    with torch.cuda.stream(s):
        for _ in range(50):
            x.add_(1.0)
        xs.dropout(executor, x, 0.0, 1, 0, y)
        total = y.sum()
    s.synchronize()
    assert total.item() == 50.0 * (1 << 22)
    assert executor.launch_count() > before


def test_same_inputs_same_bits(executor):
    """Nothing depends on the order in which blocks finish."""
    x, wg, wu = ffn_problem(1500, 264, 200, bf16)
    gate, up = (x @ wg.t()), (x @ wu.t())
    dy = rand(1, 1500, 200, dtype=bf16)

    def once():
        dx, a, b = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
        xs.gated_ffn_backward(executor, dy, x, wg, wu, gate, up, dx, a, b)
        m, r = torch.zeros(1500, device="cuda"), torch.ones(1500, device="cuda")
        dn, dw, db = torch.empty_like(x), torch.empty(264, device="cuda"), torch.empty(264, device="cuda")
        xs.layer_norm_backward(executor, x, x, None, m, r, dn, dw, db)
        return dx, a, b, dn, dw, db

    first = once()
    for _ in range(5):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


def test_c_entries_refuse_bad_arguments(executor):
    L, h = _lib.lib(), executor.handle
    t = torch.zeros(64, device="cuda")
    p = t.data_ptr()

    def refused(rc, text):
        assert rc == 1 and text in L.xspmm_last_error()

    refused(L.xspmm_layer_norm_f32f32(h, 2, 0, p, 8, None, None, 1e-5, p, 8, None, None), b"cols positive")
    refused(L.xspmm_layer_norm_f32f32(h, 2, 8, p, 7, None, None, 1e-5, p, 8, None, None), b"row stride of x")
    refused(L.xspmm_layer_norm_f32f32(h, 2, 8, p, 8, None, None, -1.0, p, 8, None, None), b"eps")
    refused(L.xspmm_layer_norm_f32f32(h, 2, 8, None, 8, None, None, 1e-5, p, 8, None, None), b"null x")
    refused(L.xspmm_layer_norm_f32f32(h, 2, 8, p + 2, 8, None, None, 1e-5, p, 8, None, None), b"not aligned")
    refused(L.xspmm_layer_norm_backward_f32f32(h, 2, 8, p, 8, p, 8, None, None, p, p, 8, None, None),
            b"null mean or rstd")
    refused(L.xspmm_dropout_f32(h, -1, p, None, 0.5, 0, 0, p), b"negative")
    refused(L.xspmm_dropout_f32(h, 4, p, None, 1.5, 0, 0, p), b"[0, 1]")
    refused(L.xspmm_gated_ffn_f16(h, 1, 8, 8, 9, p, 8, p, 8, p, 8, p, 8, None, None), b"activation")
    refused(L.xspmm_gated_ffn_f16(h, 1, 8, -8, 0, p, 8, p, 8, p, 8, p, 8, None, None), b"negative")
    refused(L.xspmm_gated_ffn_backward_f16(h, 1, 8, 8, 0, p, 8, p, 8, p, 8, p, 8, p, p, None, 8, p, None),
            b"both or neither")
