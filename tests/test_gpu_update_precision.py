"""GPU tests of the orthogonalised update's error before the rounding of its output, which is 2^-12 of it in fp16 and
would hide one of 1e-4.

The rounding of the result is independent of the error e before it, so |y - ref|^2 = |round(ref) - ref|^2 + |e|^2, from
which e follows for thousands of elements and more.

Tolerance. A sum of products is made of runs of 128 terms, 8 additions of which are truncated, by half a step of 2^-23 on
average: 2^-21 of the sum; operands of 22 bits and roundings to nearest are below that. A step has three products. It
hands on a relative error of a singular value s times s p'(s) / p(s), at most 1.61 in magnitude for s up to 1.1, and the
few values above that once by at most 5: five steps add up to (1.61^5 - 1) / 0.61 = 16.1 steps' errors. 16.1 * 3 * 2^-21
= 2.3e-5. (Sums left whole in the tensor core's accumulator: 5e-5 and 9.7e-5 at the two largest sizes. The high parts of
the operands alone: above 1e-3.)
"""
import pytest
import torch

import xspmm_b200 as xs
from test_gpu_orthogonalize import bf16, check, f16, rand, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("strong", [False, True])
@pytest.mark.parametrize("rows,cols", [(128, 128), (100, 250), (300, 500), (512, 2048), (3000, 700), (1341, 8144), (4096, 4096),
                                       (11008, 4096)])
def test_error_before_the_rounding(executor, rows, cols, strong):
    g = rand(rows + cols, rows, cols)
    if strong:
        g += 2.0 * rand(1, rows, 4) @ rand(2, 4, cols)
    y = torch.empty(rows, cols, dtype=f16, device="cuda")
    xs.orthogonalize(executor, g, y)
    ref = reference(g)
    square = lambda v: (v * v).sum().item()  # noqa: E731
    rounding = square(ref.half().double() - ref)
    error = max(0.0, square(y.double() - ref) - rounding) / square(ref)
    assert error ** 0.5 <= 16.1 * 3 * 2.0 ** -21, error ** 0.5


@pytest.mark.parametrize("rows,cols", [(100, 100), (64, 200), (300, 200), (200, 700), (900, 260)])
@pytest.mark.parametrize("halvings,steps", [(1, 5), (10, 5), (20, 5), (20, 16), (45, 5), (90, 5), (90, 1)])
def test_gradients_far_below_eps(executor, rows, cols, halvings, steps):
    """|g| = eps 2^-halvings: X_0 is as small, and every step multiplies it by 3.4445 until it is near 1."""
    base = rand(4, rows, cols).double()
    g = (base / torch.linalg.matrix_norm(base) * (1e-7 * 2.0 ** -halvings)).float()
    y = torch.empty(rows, cols, dtype=bf16, device="cuda")
    xs.orthogonalize(executor, g, y, steps=steps)
    check(y, reference(g, steps))
