"""GPU tests of the 8-bit product and the orthogonalised update at sizes whose products give a CTA (pair) several tiles
one after the other, and whole tiles next to ones whose sum is split: what a tile leaves behind (accumulators, the ring
of stages, staging pieces) is taken up by the next.

On 148 SMs, 74 pairs: the symmetric products of 3100 x 3100 are 74 whole tiles and 17 split by four, its others 221
tiles; 2300 x 3100 ends in 148 whole tiles and 5 split; 100 x 40000 gives 148 single CTAs 250 tiles; 6000 x 1200 is the
tall form. The 8-bit products are 120 tiles, 74 whole ones and 10 split, and for 100 rows 148 whole ones and 2 split.
Tolerances are those of the operators' own tests.
"""
import pytest
import torch

import xspmm_b200 as xs
from test_gpu_int8 import check as check_int8
from test_gpu_int8 import whole
from test_gpu_orthogonalize import check, rand, reference

pytestmark = pytest.mark.gpu

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("rows,cols", [(3100, 3100), (2300, 3100), (100, 40000), (6000, 1200), (1203, 5999)])
@pytest.mark.parametrize("tx,ty", [(f32, f16), (bf16, bf16)])
def test_update(executor, rows, cols, tx, ty):
    g = rand(rows + cols, rows, cols, dtype=tx, scale=1e-2)
    buf = torch.full((rows * cols + 64,), 7.0, dtype=ty, device="cuda")
    y = buf[:rows * cols].view(rows, cols)
    xs.orthogonalize(executor, g, y)
    check(y, reference(g))
    assert (buf[rows * cols:] == 7.0).all()
    again = torch.empty_like(y)
    xs.orthogonalize(executor, g, again)
    assert torch.equal(y, again)


@pytest.mark.parametrize("rows,K,F", [(2500, 2048, 3000), (2500, 2048, 3001), (1300, 8192, 3400), (100, 8192, 38200)])
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("biased", [True, False])
def test_linear_int8(executor, rows, K, F, dtype, biased):
    x, w = whole(1, rows, K), whole(2, F, K)
    xs_, ws, bias = rand(3, rows).abs() / 64, rand(4, F).abs() / (64 * K ** 0.5), rand(5, F)
    buf = torch.full((rows * F + 64,), 7.0, dtype=dtype, device="cuda")
    y = buf[:rows * F].view(rows, F)
    xs.linear_int8(executor, x, xs_, w, ws, y, bias=bias if biased else None)
    check_int8(y, x, xs_, w, ws, bias if biased else None)
    assert (buf[rows * F:] == 7.0).all()


@pytest.mark.parametrize("rows", [40, 300])
def test_padded_operands_are_read_in_place(executor, rows):
    """Slices of rows padded to 16 bytes give the same product with one launch less: nothing is copied."""
    K, F = 1021, 531
    x, w, s, ws = whole(1, rows, K), whole(2, F, K), rand(3, rows), rand(4, F)
    launches, outs = [], []
    for a, b in ((x, w), (torch.nn.functional.pad(x, (0, 3))[:, :K], torch.nn.functional.pad(w, (0, 3))[:, :K])):
        y = torch.empty(rows, F, dtype=f16, device="cuda")
        executor.reset_launch_count()
        xs.linear_int8(executor, a, s, b, ws, y)
        launches.append(executor.launch_count())
        outs.append(y)
    assert torch.equal(*outs) and launches[1] == launches[0] - 1
