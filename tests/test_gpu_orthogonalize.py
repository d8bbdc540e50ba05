"""GPU tests of the orthogonalised update against the iteration in 64 bits.

Tolerances. An error of X along a direction of small singular value grows by at most a = 3.4445 a step, 485 times
in five; along the others the polynomial's slope is at most 4 where it is steepest and the singular values do not
stay there. A step's own error is that of 22-bit operands and fp32 sums, relative to the operands: 4 * 2^-21. So
the whole of y is within R = 485 * 4 * 2^-21 of itself in the 2-norm, on top of the rounding to its type, and no
single element is off by more than 16 times that of the root of the mean square.
"""
import pytest
import torch

import xspmm_b200 as xs

pytestmark = pytest.mark.gpu

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32
U = {f16: 2.0 ** -11, bf16: 2.0 ** -8}
R = 485 * 4 * 2.0 ** -21
TYPES = [(f16, f16), (bf16, bf16), (f32, f16), (f32, bf16)]
A, B, C = 3.4445, -4.7750, 2.0315


def rand(seed, *shape, dtype=f32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def reference(g, steps=5, eps=1e-7):
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x) + eps)
    for _ in range(steps):
        if x.shape[0] <= x.shape[1]:
            a = x @ x.t()
            x = A * x + B * (a @ x) + C * (a @ (a @ x))
        else:
            a = x.t() @ x
            x = A * x + B * (x @ a) + C * ((x @ a) @ a)
    return x


def check(y, ref):
    off, u = (y.double() - ref), U[y.dtype]
    norm = torch.linalg.vector_norm(ref).item()
    rms = norm / max(ref.numel(), 1) ** 0.5
    assert torch.isfinite(y).all()
    assert torch.linalg.vector_norm(off).item() <= 1.01 * (u + R) * norm
    tiny = 2.0 ** -25 if y.dtype == f16 else 0.0
    assert (off.abs() <= 1.01 * (u * ref.abs() + 16 * R * rms) + tiny).all()


SIZES = [(1, 1), (1, 300), (300, 1), (2, 3), (16, 16), (7, 130), (130, 7), (64, 64), (128, 128), (127, 128), (100, 77), (128, 1000),
         (1021, 90), (129, 129), (200, 300), (256, 256), (301, 517), (640, 384), (513, 1100), (1024, 1024), (1500, 2100)]


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_update(executor, rows, cols, tx, ty):
    g = rand(rows * 7 + cols, rows, cols, dtype=tx, scale=1e-2)
    buf = torch.full((rows * cols + 64,), 7.0, dtype=ty, device="cuda")
    y = buf[:rows * cols].view(rows, cols)
    xs.orthogonalize(executor, g, y)
    check(y, reference(g))
    assert (buf[rows * cols:] == 7.0).all()


@pytest.mark.parametrize("rows,cols", [(96, 96), (200, 700), (900, 260)])
@pytest.mark.parametrize("spread", [1.0, 1e-2, 1e-4])
def test_singular_values(executor, rows, cols, spread):
    """Singular values from 1 down to `spread`: the largest fall into [0.68, 1.21] and small ones grow by a^5."""
    m = min(rows, cols)
    u, _ = torch.linalg.qr(rand(1, rows, m).double())
    v, _ = torch.linalg.qr(rand(2, cols, m).double())
    s = torch.logspace(0, torch.log10(torch.tensor(spread)).item(), m, dtype=torch.float64, device="cuda")
    g = ((u * s) @ v.t()).float()
    y = torch.empty(rows, cols, dtype=f16, device="cuda")
    xs.orthogonalize(executor, g, y)
    check(y, reference(g))


@pytest.mark.parametrize("steps", [0, 1, 2, 8])
def test_steps(executor, steps):
    for rows, cols in ((90, 140), (300, 200)):
        g = rand(3, rows, cols, dtype=bf16)
        y = torch.empty_like(g)
        xs.orthogonalize(executor, g, y, steps=steps)
        check(y, reference(g, steps))


def test_scale_of_the_gradient(executor):
    """The result does not depend on g's scale down to eps; squares that leave fp32's range do not matter. A
    gradient of the size of eps is damped, one of zeros gives zeros."""
    base = rand(4, 150, 260)
    for scale in (1e-25, 1e-10, 1.0, 1e25):
        for g in (base * scale, (base * scale).t().contiguous()):
            eps = 1e-7 if scale >= 1.0 else 0.0
            y = torch.empty(g.shape, dtype=f16, device="cuda")
            xs.orthogonalize(executor, g, y, eps=eps)
            check(y, reference(g, eps=eps))
    g = base / torch.linalg.matrix_norm(base.double()).float() * 1e-7
    y = torch.empty(g.shape, dtype=f16, device="cuda")
    xs.orthogonalize(executor, g, y)
    check(y, reference(g))
    for rows, cols in ((5, 5), (150, 260)):
        y = torch.full((rows, cols), 7.0, dtype=bf16, device="cuda")
        xs.orthogonalize(executor, torch.zeros(rows, cols, device="cuda"), y)
        assert not y.any()


@pytest.mark.parametrize("rows,cols", [(40, 40), (150, 260), (260, 150), (700, 400)])
def test_a_single_large_entry(executor, rows, cols):
    """All of the norm in one entry, the others 2^-20 of it."""
    g = rand(5, rows, cols, scale=2.0 ** -20)
    g[rows // 2, cols // 3] = 1.0
    y = torch.empty(rows, cols, dtype=f16, device="cuda")
    xs.orthogonalize(executor, g, y)
    check(y, reference(g))


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("pad", [1, 8])
def test_strides(executor, tx, ty, pad):
    for rows, cols in ((60, 72), (180, 136), (200, 331)):
        g = rand(6, rows, cols + 2 * pad, dtype=tx)[:, pad:pad + cols]
        buf = torch.full((rows, cols + 2 * pad), 7.0, dtype=ty, device="cuda")
        y = buf[:, pad:pad + cols]
        xs.orthogonalize(executor, g, y)
        check(y, reference(g))
        assert (buf[:, :pad] == 7.0).all() and (buf[:, pad + cols:] == 7.0).all()


def test_in_place_and_empty(executor):
    for rows, cols in ((100, 100), (300, 170)):
        g = rand(7, rows, cols, dtype=bf16)
        y = torch.empty_like(g)
        xs.orthogonalize(executor, g, y)
        xs.orthogonalize(executor, g, g)
        assert torch.equal(g, y)
    xs.orthogonalize(executor, g[:0], y[:0])
    xs.orthogonalize(executor, g[:, :0], y[:, :0])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("rows,cols", [(50, 50), (200, 300)])
def test_not_finite(executor, rows, cols, bad):
    g = rand(8, rows, cols)
    g[3, 4] = bad
    y = torch.zeros(rows, cols, dtype=f16, device="cuda")
    xs.orthogonalize(executor, g, y)
    assert torch.isnan(y).all()


@pytest.mark.parametrize("rows,cols", [(128, 96), (400, 530)])
def test_streams_graphs_and_repeats(executor, rows, cols):
    g = rand(9, rows, cols, dtype=f16)
    first, other = torch.empty_like(g), torch.empty_like(g)
    xs.orthogonalize(executor, g, first)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        xs.orthogonalize(executor, g, other)
    side.synchronize()
    assert torch.equal(first, other)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], [torch.zeros_like(g), torch.zeros_like(g)]
    for graph, out in zip(graphs, outs):
        with torch.cuda.graph(graph):
            xs.orthogonalize(executor, g, out)
    g.copy_(rand(10, rows, cols, dtype=f16))
    for graph in graphs:
        graph.replay()
    xs.orthogonalize(executor, g, first)
    torch.cuda.synchronize()
    check(first, reference(g))
    for out in outs:
        assert torch.equal(first, out)
