"""GPU tests of rows in 8-bit integers and their product.

Quantisation is exact: q and scale are compared for equality with whole-number arithmetic. The product's sum is
exact; the result takes a rounding of the sum to fp32, two of its products with the scales, one of the bias and
one to y's type: 4 * 2^-24 of the terms' magnitudes and U[T] of the result.
"""
import pytest
import torch

import xspmm_b200 as xs

pytestmark = pytest.mark.gpu

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32
U = {f16: 2.0 ** -11, bf16: 2.0 ** -8, f32: 2.0 ** -24}
TINY = {f16: 2.0 ** -25, bf16: 2.0 ** -134, f32: 2.0 ** -149}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rand(seed, *shape, dtype=f32, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def whole(seed, *shape, low=-128, high=128):
    return torch.randint(low, high, shape, generator=gen(seed), device="cuda", dtype=torch.int8)


def quantized(x):
    """q by comparing whole multiples: 127 |x| / most to the nearest, ties to even. 64-bit products of fp32
    numbers with 8-bit ones are exact; the quotient of two of them is never within 2^-27 of a border it does not
    hit, so 64 bits decide it."""
    x = x.double()
    most = x.abs().amax(1, keepdim=True) if x.shape[1] else torch.zeros(x.shape[0], 1, dtype=torch.float64, device="cuda")
    q = torch.where(most > 0, torch.round(127.0 * x / torch.where(most > 0, most, torch.ones_like(most))), torch.zeros_like(x))
    return q.to(torch.int8), (most[:, 0] / 127.0).float()  # 64 bits hold the fp32 quotient's rounding


@pytest.mark.parametrize("dtype", [f16, bf16, f32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (257, 128), (64, 129), (33, 1000), (9, 1021), (5, 16384),
                                       (2, 20001), (1000, 24), (20000, 40), (4, 8190), (700, 2048), (3, 40000)])
def test_quantize(executor, rows, cols, dtype):
    x = rand(rows + cols, rows, cols, dtype=dtype, scale=3.0)
    q, scale = torch.full((rows, cols), 77, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    xs.quantize_rows(executor, x, q, scale)
    rq, rs = quantized(x)
    assert torch.equal(q, rq) and torch.equal(scale, rs)


@pytest.mark.parametrize("dtype", [f16, bf16, f32])
def test_quantize_borders(executor, dtype):
    """Quotients on a border (most a multiple of 127: ties) and as near to one as the type gets."""
    most = torch.tensor([127.0, 254.0, 2.0 ** -10 * 127], device="cuda")[:, None]
    half = (torch.arange(-127, 127, device="cuda") + 0.5)[None, :] * most / 127
    x = torch.cat((most, half), 1).to(dtype)
    up = torch.nextafter(x.float(), torch.full_like(x.float(), 1e30)) if dtype == f32 else x
    for v in (x, up, -x, rand(5, 4000, 64, dtype=dtype)):
        v = v.contiguous()
        q, scale = torch.empty(v.shape, dtype=torch.int8, device="cuda"), torch.empty(v.shape[0], device="cuda")
        xs.quantize_rows(executor, v, q, scale)
        rq, rs = quantized(v)
        assert torch.equal(q, rq) and torch.equal(scale, rs)


def test_quantize_extremes(executor):
    """Zeros, subnormals, the largest numbers, infinities and NaN, each row by itself."""
    x = rand(1, 9, 200, dtype=f32)
    x[1] = 0.0
    x[2] *= 1e-40
    x[3] *= 1e37
    x[4, 5] = float("inf")
    x[5, 7] = float("nan")
    x[6], x[6, 199] = 0.0, 2.0 ** -149
    x[7, 0] = 3.4028234663852886e38
    q, scale = torch.full(x.shape, 9, dtype=torch.int8, device="cuda"), torch.empty(9, device="cuda")
    xs.quantize_rows(executor, x, q, scale)
    fine = [0, 1, 2, 3, 6, 7, 8]
    rq, rs = quantized(x[fine])
    assert torch.equal(q[fine], rq) and torch.equal(scale[fine], rs)
    assert torch.isnan(scale[[4, 5]]).all() and not q[[4, 5]].any()
    assert scale[1].item() == 0.0 and not q[1].any()
    empty = torch.empty(4, 0, device="cuda")
    s = torch.ones(4, device="cuda")
    xs.quantize_rows(executor, empty, empty.to(torch.int8), s)
    assert not s.any()
    xs.quantize_rows(executor, x[:0], q[:0], scale[:0])


@pytest.mark.parametrize("dtype", [f16, bf16, f32])
@pytest.mark.parametrize("pad", [1, 4, 16])
def test_quantize_strides(executor, dtype, pad):
    for cols in (128, 1000, 37):
        x = rand(2, 50, cols + 2 * pad, dtype=dtype)[:, pad:pad + cols]
        buf = torch.full((50, cols + 3 * pad), 77, dtype=torch.int8, device="cuda")
        scale = torch.empty(50, device="cuda")
        xs.quantize_rows(executor, x, buf[:, pad:pad + cols], scale)
        rq, rs = quantized(x)
        assert torch.equal(buf[:, pad:pad + cols], rq) and torch.equal(scale, rs)
        assert (buf[:, :pad] == 77).all() and (buf[:, pad + cols:] == 77).all()


def exact_sum(x, w):
    return x.double() @ w.double().t()  # below 2^31 in magnitude: exact in 64 bits


def check(y, x, xs_, w, ws, bias):
    t = exact_sum(x, w) * xs_.double()[:, None] * ws.double()
    b = torch.zeros_like(ws).double() if bias is None else bias.double()
    ref = t + b
    err = 4 * 2.0 ** -24 * (t.abs() + b.abs())
    tol = 1.01 * (err + U[y.dtype] * ref.abs()) + TINY[y.dtype]
    # past the type's largest number by more than half a step (and the error) the result is infinite
    last = torch.finfo(y.dtype).max
    over = ref.abs() - err > last * (1.0 + U[y.dtype])
    assert torch.equal(y[over].double(), torch.sign(ref[over]) * float("inf"))
    inside = ref.abs() + err < last
    assert torch.isfinite(y[inside]).all()
    assert ((y.double() - ref).abs() <= tol)[inside].all(), f"off by {(y.double() - ref).abs().max().item():.3e}"


SIZES = [(1, 1, 1), (1, 4096, 500), (3, 16, 16), (8, 33, 70), (16, 1000, 1000), (17, 64, 32), (33, 1021, 77), (64, 4096, 130),
         (128, 128, 128), (129, 256, 300), (301, 1021, 531), (257, 32, 2000), (1000, 48, 24), (2100, 160, 96), (300, 11008, 64),
         (5, 70000, 9), (40, 70000, 9), (640, 2048, 513), (4000, 16, 8)]


@pytest.mark.parametrize("dtype", [f16, bf16, f32])
@pytest.mark.parametrize("rows,K,F", SIZES)
def test_linear(executor, rows, K, F, dtype):
    x, w = whole(rows, rows, K), whole(K, F, K)
    xs_ = rand(3, rows).abs() / 64
    ws = rand(4, F).abs() / (64 * K ** 0.5)
    for bias in (None, rand(5, F)):
        buf = torch.full((rows * F + 64,), 7.0, dtype=dtype, device="cuda")
        y = buf[:rows * F].view(rows, F)
        xs.linear_int8(executor, x, xs_, w, ws, y, bias=bias)
        check(y, x, xs_, w, ws, bias)
        assert (buf[rows * F:] == 7.0).all()


@pytest.mark.parametrize("rows,F", [(2, 20), (200, 40)])
def test_linear_largest_sums(executor, rows, F):
    """131071 products of -128 by -128 stay within 32 bits; one column more is refused."""
    K = 131071
    x, w = torch.full((rows, K), -128, dtype=torch.int8, device="cuda"), torch.full((F, K), -128, dtype=torch.int8, device="cuda")
    x[1], w[3] = 127, 127
    xs_, ws = torch.ones(rows, device="cuda"), torch.ones(F, device="cuda")
    y = torch.empty(rows, F, device="cuda")
    xs.linear_int8(executor, x, xs_, w, ws, y)
    check(y, x, xs_, w, ws, None)
    more = torch.zeros(rows, K + 1, dtype=torch.int8, device="cuda")
    with pytest.raises(ValueError, match="at most"):
        xs.linear_int8(executor, more, xs_, more, xs_, y)


@pytest.mark.parametrize("dtype", [f16, bf16, f32])
@pytest.mark.parametrize("rows", [3, 40, 200, 520])
@pytest.mark.parametrize("pad", [1, 8, 16])
def test_linear_strides(executor, rows, pad, dtype):
    """Slices of columns of wider tensors, aligned and not; nothing is written outside."""
    K, F = 272, 96
    x, w = whole(1, rows, K + 2 * pad)[:, pad:pad + K], whole(2, F, K + pad)[:, :K]
    xs_, ws, bias = rand(3, rows), rand(4, F), rand(5, F)
    buf = torch.full((rows, F + 2 * pad), 7.0, dtype=dtype, device="cuda")
    y = buf[:, pad:pad + F]
    xs.linear_int8(executor, x, xs_, w, ws, y, bias=bias)
    check(y, x, xs_, w, ws, bias)
    assert (buf[:, :pad] == 7.0).all() and (buf[:, pad + F:] == 7.0).all()


@pytest.mark.parametrize("rows", [4, 300])
def test_linear_row_with_an_infinity(executor, rows):
    """A quantised row with an infinity makes its own products NaN, and no others."""
    x = rand(1, rows, 64, dtype=f16)
    x[2, 3] = float("inf")
    q, s = torch.empty(rows, 64, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    xs.quantize_rows(executor, x, q, s)
    w, ws = whole(2, 24, 64), rand(3, 24)
    y = torch.empty(rows, 24, dtype=f16, device="cuda")
    xs.linear_int8(executor, q, s, w, ws, y)
    assert torch.isnan(y[2]).all()
    y[2] = 0.0
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("rows", [3, 200])
def test_linear_of_nothing(executor, rows):
    ws, bias = rand(1, 24), rand(2, 24)
    y = torch.empty(rows, 24, dtype=bf16, device="cuda")
    none = torch.empty(rows, 0, dtype=torch.int8, device="cuda")
    xs.linear_int8(executor, none, rand(3, rows), torch.empty(24, 0, dtype=torch.int8, device="cuda"), ws, y, bias=bias)
    assert torch.equal(y, bias.bfloat16().expand(rows, 24))
    xs.linear_int8(executor, none, rand(3, rows), torch.empty(24, 0, dtype=torch.int8, device="cuda"), ws, y)
    assert not y.any()
    q = whole(4, rows, 8)
    xs.linear_int8(executor, q[:0], ws[:0], whole(5, 24, 8), ws, y[:0])
    xs.linear_int8(executor, q, rand(3, rows), q[:0], ws[:0], torch.empty(rows, 0, dtype=bf16, device="cuda"))


@pytest.mark.parametrize("rows", [5, 100, 700])
def test_streams_and_graphs(executor, rows):
    """Quantise and multiply on another stream and from a captured graph, on new inputs: the same numbers."""
    K, F = 1000, 1040
    x, w, ws = rand(1, rows, K, dtype=bf16), whole(2, F, K), rand(3, F)

    def call():
        q, s = torch.empty(rows, K, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
        y = torch.empty(rows, F, dtype=bf16, device="cuda")
        xs.quantize_rows(executor, x, q, s)
        xs.linear_int8(executor, q, s, w, ws, y)
        return q, s, y

    first = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(call())
    x.mul_(-0.5)
    for g in graphs:
        g.replay()
    again = call()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(again, out))
    check(again[2], again[0], again[1], w, ws, None)
