"""GPU tests of the gated feed-forward block at gates far from 0, against the formulas in 64 bits, on every
path: a few rows, tiles of one CTA and of a pair, tiles whose sum is split; gradients in one pass over the
rows, and by slopes and products.

The gates are put in place exactly: x has a column of ones and w_gate the gate there. Tolerances: e^-v is
2^(-v log2 e), whose exponent carries a rounding of 2^-24 of itself, so its relative error is within
(|v| + 16) * 2^-23 with the exponential's own; as much again covers the products after it. Past e^87.3 the
fp32 quotient may be 0 instead of a value below |v| * 2^-126. On top comes half a unit of the output type
(U), or of its subnormals (TINY).
"""
import pytest
import torch

import xspmm_b200 as xs

pytestmark = pytest.mark.gpu

f16, bf16 = torch.float16, torch.bfloat16
U = {f16: 2.0 ** -11, bf16: 2.0 ** -8}
TINY = {f16: 2.0 ** -25, bf16: 2.0 ** -134}
GATES = {bf16: [-1e20, -1e4, -120.0, -100.0, -88.0, -87.0, -60.0, -50.0, -42.0, -41.0, -40.0, -20.0, -6.0, -1.0,
                0.0, 1.0, 6.0, 41.0, 42.0, 50.0, 1e4, 1e20],
         f16: [-6e4, -1e4, -120.0, -100.0, -60.0, -50.0, -42.0, -41.0, -40.0, -20.0, -10.0, -6.0, -1.0, 0.0, 1.0,
               6.0, 41.0, 50.0]}
PATHS = [(3, 64), (3, 61), (100, 64), (200, 64), (200, 4096)]  # rows, K


def gates(n, dtype, odd=None):
    """n gates; `odd`, if given, at every 37th place."""
    v = torch.tensor([GATES[dtype][i % len(GATES[dtype])] for i in range(n)], device="cuda").to(dtype)
    if odd is not None:
        v[5::37] = odd
    return v


def silu(v):
    v = v.clamp(min=-1e6)  # 0 there, in 64 bits too
    return v * torch.sigmoid(v)


def silu_slope(v):
    v = v.clamp(-1e6, 1e6)
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def sigmoid_error(v):
    return torch.sigmoid(v) * (v.abs().clamp(max=100) + 16) * 2.0 ** -22


def silu_error(v):
    return v.abs().clamp(max=1e30) * sigmoid_error(v) + 100 * 2.0 ** -126


def silu_slope_error(v):
    """1 - s carries s's error, and v * (1 - s) no more than at |v| = 100, where s is 0 or 1."""
    return (1 + v.abs().clamp(max=100)) * (sigmoid_error(v) + 2.0 ** -126)


def close(got, ref, err, what):
    T = got.dtype
    off, tol = (got.double() - ref).abs(), 1.01 * (err + U[T] * ref.abs()) + TINY[T]
    same = (got.double() == ref) | (off <= tol)
    assert bool(same.all()), (what, got[~same][:4], ref[~same][:4])


def forward(executor, rows, K, gate, up, act="silu"):
    """y and the projections of rows whose gates are `gate` and whose up projection is `up`."""
    F, dtype = gate.numel(), gate.dtype
    x = torch.zeros(rows, K, dtype=dtype, device="cuda")
    wg, wu = torch.zeros(F, K, dtype=dtype, device="cuda"), torch.zeros(F, K, dtype=dtype, device="cuda")
    x[:, 3] = 1.0
    wg[:, 3] = gate
    wu[:, 3] = up
    y, g, u = (torch.empty(rows, F, dtype=dtype, device="cuda") for _ in range(3))
    xs.gated_ffn(executor, x, wg, wu, y, act, g, u)
    return y, g, u


@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("rows,K", PATHS)
def test_silu_far_from_zero(executor, rows, K, dtype):
    """An up projection of 2^14 shows what a sigmoid that does not fall to 0 would leave."""
    v = gates(200, dtype)
    up = 2.0 ** (14 if dtype == bf16 else 4)
    y, g, u = forward(executor, rows, K, v, up)
    assert torch.equal(g, v.expand_as(g)) and bool((u == up).all())
    v = v.double()
    close(y, (silu(v) * up).expand(rows, -1), silu_error(v) * up, "y")
    assert bool((y[:, v < -110] == 0).all())


@pytest.mark.parametrize("rows,K", PATHS)
def test_silu_of_a_projection_that_overflows(executor, rows, K):
    """A gate that passes fp32's range downwards gives 0, as every large negative gate does."""
    F = 72
    x = torch.zeros(rows, K, dtype=bf16, device="cuda")
    wg, wu = torch.zeros(F, K, dtype=bf16, device="cuda"), torch.zeros(F, K, dtype=bf16, device="cuda")
    x[:, 0], x[:, 1] = 3e38, 1.0
    wg[::5, 0], wg[:, 1], wu[:, 1] = -4.0, 1.0, 2.0
    y, gate = (torch.empty(rows, F, dtype=bf16, device="cuda") for _ in range(2))
    xs.gated_ffn(executor, x, wg, wu, y, "silu", gate)
    assert bool((gate[:, ::5] == -torch.inf).all())
    assert bool((y[:, ::5] == 0).all())
    one = silu(torch.ones((), dtype=torch.float64, device="cuda")) * 2
    rest = [f for f in range(F) if f % 5]
    close(y[:, rest], one.expand(rows, len(rest)), 2.0 ** -18, "beside them")


@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("rows,K", PATHS)
def test_a_gate_that_is_not_a_number_stays_alone(executor, rows, K, dtype):
    v = gates(200, dtype, odd=torch.nan)
    y, _, _ = forward(executor, rows, K, v, 1.0)
    bad = torch.isnan(v)
    assert bool(torch.isnan(y[:, bad]).all())
    v = v[~bad].double()
    close(y[:, ~bad], silu(v).expand(rows, -1), silu_error(v), "y")


@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("n", [64, 128, 191, 200])
@pytest.mark.parametrize("odd", [None, torch.inf, -torch.inf, torch.nan])
def test_silu_gradient_far_from_zero(executor, n, dtype, odd):
    """x is the identity, so that dw_gate and dw_up are dgate and dup themselves, transposed. An infinite gate
    has the slope of the limit, 0 or 1."""
    eye = torch.eye(n, dtype=dtype, device="cuda")
    zero = torch.zeros_like(eye)
    gate = gates(n * n, dtype, odd).view(n, n)
    dy, up = torch.full_like(eye, 0.5), torch.full_like(eye, 8.0)
    dx, dwg, dwu = torch.empty_like(eye), torch.empty_like(eye), torch.empty_like(eye)
    xs.gated_ffn_backward(executor, dy, eye, zero, zero, gate, up, dx, dwg, dwu)
    if odd is not None and odd != odd:  # every sum over the rows that holds it; nothing else
        cols = torch.isnan(gate).any(0)
        assert bool(torch.isnan(dwg[cols]).all()) and bool(torch.isnan(dwu[cols]).all())
        gate, dwg, dwu = gate[:, ~cols], dwg[~cols], dwu[~cols]
    v = gate.double().t()
    close(dwg, 4.0 * silu_slope(v), 4.0 * silu_slope_error(v), "dgate")
    keep = (v != torch.inf).all(1)
    dwu, v = dwu[keep], v[keep]
    close(dwu, 0.5 * silu(v), 0.5 * silu_error(v), "dup")


# ---- gelu -------------------------------------------------------------------------------------------
# gelu = v * erfc(-v / sqrt 2) / 2. The tail's formula is within 2^-20 of itself with its roundings; e^(-v^2 / 2)
# carries the roundings of its argument (three of 2^-24 times v^2 / 2) and the exponential's own. (v^2 + 16) * 2^-22
# of each term covers them with the products after it. Values below 16 * 2^-126 may be 0.

TAIL = {bf16: [-1e20, -1e4, -100.0, -16.0, -12.0, -11.0, -10.0, -9.0, -8.0, -7.0, -6.0, -5.5, -5.0, -4.5, -4.0, -3.0,
               -2.0, -1.0, -0.25, 0.0, 0.5, 1.0, 3.0, 6.0, 20.0, 1e4],
        f16: [-6e4, -100.0, -16.0, -8.0, -6.5, -6.0, -5.75, -5.5, -5.25, -5.0, -4.75, -4.5, -4.25, -4.0, -3.0, -2.0,
              -1.0, 0.0, 1.0, 3.0, 6.0]}


def tail(n, dtype):
    return torch.tensor([TAIL[dtype][i % len(TAIL[dtype])] for i in range(n)], device="cuda").to(dtype)


def gelu_terms(v):
    """gelu(v), its slope's two terms, and the relative error of each."""
    v = v.clamp(min=-1e3)
    half = 0.5 * torch.special.erfc(-v * 0.5 ** 0.5)
    c = v.clamp(max=1e3)
    return v * half, half, c * torch.exp(-0.5 * c * c) * (2 * torch.pi) ** -0.5, (v.abs().clamp(max=20) ** 2 + 16) * 2.0 ** -22


@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("rows,K", PATHS)
def test_gelu_of_negative_gates(executor, rows, K, dtype):
    v = tail(200, dtype)
    y, _, _ = forward(executor, rows, K, v, 1024.0, "gelu")
    value, _, _, rel = gelu_terms(v.double())
    close(y, (1024 * value).expand(rows, -1), 1024 * (value.abs() * rel + 16 * 2.0 ** -126), "y")


@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("n", [64, 128, 191, 200])
@pytest.mark.parametrize("odd", [None, torch.inf, -torch.inf])
def test_gelu_gradient_of_negative_gates(executor, n, dtype, odd):
    eye = torch.eye(n, dtype=dtype, device="cuda")
    zero = torch.zeros_like(eye)
    gate = tail(n * n, dtype)
    if odd is not None:
        gate[5::37] = odd
    gate = gate.view(n, n)
    dy, up = torch.full_like(eye, 64.0), torch.full_like(eye, 64.0)
    dx, dwg, dwu = torch.empty_like(eye), torch.empty_like(eye), torch.empty_like(eye)
    xs.gated_ffn_backward(executor, dy, eye, zero, zero, gate, up, dx, dwg, dwu, activation="gelu")
    v = gate.double().t()
    value, half, bell, rel = gelu_terms(v)
    close(dwg, 4096 * (half + bell), 4096 * ((half + bell.abs()) * rel + 16 * 2.0 ** -126), "dgate")
    keep = (v != torch.inf).all(1)
    close(dwu[keep], 64 * value[keep], 64 * (value.abs() * rel + 16 * 2.0 ** -126)[keep], "dup")


# ---- sigmoid ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [f16, bf16])
@pytest.mark.parametrize("n", [64, 191, 200])
@pytest.mark.parametrize("odd", [None, torch.inf, -torch.inf])
def test_sigmoid_gradient_far_from_zero(executor, n, dtype, odd):
    """s (1 - s) falls off as e^-|v| on both sides. The errors are those of silu's sigmoid."""
    v = [0.0, 1.0, 3.0, 6.0, 8.0, 10.0, 11.0, 12.0, 14.0, 16.0, 18.0, 20.0, 30.0, 60.0, 100.0, 6e4]
    v = torch.tensor((v + [-a for a in v]) * (n * n // 32 + 1), device="cuda")[:n * n].to(dtype)
    if odd is not None:
        v[5::37] = odd
    eye = torch.eye(n, dtype=dtype, device="cuda")
    zero = torch.zeros_like(eye)
    dy, up = torch.full_like(eye, 64.0), torch.full_like(eye, 64.0)
    dx, dwg, dwu = torch.empty_like(eye), torch.empty_like(eye), torch.empty_like(eye)
    xs.gated_ffn_backward(executor, dy, eye, zero, zero, v.view(n, n), up, dx, dwg, dwu, activation="sigmoid")
    v = v.view(n, n).t().double()
    s, c = torch.sigmoid(v), torch.sigmoid(-v)
    rel = (v.abs().clamp(max=100) + 16) * 2.0 ** -22
    close(dwg, 4096 * s * c, 4096 * (s * c * rel + 2.0 ** -126), "dgate")
    close(dwu, 64 * s, 64 * (s * rel + 2.0 ** -126), "dup")
