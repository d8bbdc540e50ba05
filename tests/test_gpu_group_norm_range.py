"""GPU tests of the group norm at the ends of its range: features of large magnitude."""
import math

import pytest
import torch

import xspmm_b200 as xs
from test_gpu_group_norm import U, bf16, check_forward, f16, f32, guarded, rand, value

pytestmark = pytest.mark.gpu

# rows, cols, groups, offsets: samples by a warp, in the slots of a CTA, by a CTA in two passes, in chunks; groups wider
# than a tile; single elements; rows and widths that are no power of two, where a mean of equal values can round
SHAPES = [(1, 8, 1, None), (7, 24, 8, [0, 3, 4, 7]), (301, 84, 12, None), (600, 96, 4, [0, 600]), (3001, 24, 1, None),
          (30001, 64, 8, [0, 29999]), (9001, 300, 1, None), (500, 33, 3, list(range(0, 501, 5))), (50001, 33, 1, None),
          (40001, 200, 1, [3, 39998])]
WIDE_TYPES = [(bf16, bf16), (f32, f32), (f32, f16), (f32, bf16)]


@pytest.mark.parametrize("tx,ty", WIDE_TYPES)
@pytest.mark.parametrize("size", [1e5, 1e20, -2.5e38, 3.3e38])
@pytest.mark.parametrize("rows,cols,groups,offsets", SHAPES)
def test_constant_groups_of_any_size(executor, rows, cols, groups, offsets, size, tx, ty):
    """The mean of equal values is that value, their variance 0 and y = act(bias), in every path: no partial mean is
    rounded away from it and no sum or square leaves fp32's range."""
    c = (size * (1.0 + torch.arange(groups, device="cuda") / (64.0 * groups))).to(tx)
    x = c.repeat_interleave(cols // groups).expand(rows, cols).contiguous()
    assert torch.isfinite(x).all()
    b = rand(1, cols)
    y, buf = guarded(rows, cols, ty)
    spans = 1 if offsets is None else len(offsets) - 1
    mean, rstd = torch.empty(spans, groups, device="cuda"), torch.empty(spans, groups, device="cuda")
    dev = None if offsets is None else torch.tensor(offsets, device="cuda")
    xs.group_norm(executor, x, groups, None, b, 1e-5, y, offsets=dev, activation="silu", mean=mean, rstd=rstd)
    assert torch.equal(mean, c.float().expand(spans, groups))
    want = 1.0 / math.sqrt(torch.tensor(1e-5, dtype=f32).item())
    assert ((rstd.double() - want).abs() <= 2.0 ** -22 * want).all()
    inner = slice(0, rows) if offsets is None else slice(offsets[0], offsets[-1])
    ref = value("silu", b.double()).expand(rows, cols)[inner]
    assert ((y[inner].double() - ref).abs() <= 1.01 * (U[ty] + 2.0 ** -20) * ref.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("tx,ty", WIDE_TYPES)
@pytest.mark.parametrize("size", [1e8, 1e15])
@pytest.mark.parametrize("rows,cols,groups,offsets", SHAPES[1:])
def test_large_deviations(executor, rows, cols, groups, offsets, size, tx, ty):
    """Deviations whose squares and their sums stay in range, about a mean of their size."""
    x = rand(rows, rows, cols, dtype=tx, scale=size, shift=size)
    y, buf = guarded(rows, cols, ty)
    check_forward(executor, x, groups, None, rand(1, cols), 1e-5, y, offsets, "gelu", buf)


@pytest.mark.parametrize("tx,ty", WIDE_TYPES)
@pytest.mark.parametrize("rows,cols,groups,offsets", SHAPES[1:])
def test_squares_past_the_range(executor, rows, cols, groups, offsets, tx, ty):
    """Deviations of 1e30: the variance is infinite in fp32, so rstd is 0 and y = act(bias), not NaN."""
    x = rand(rows, rows, cols, dtype=tx, scale=1e30, shift=1e30)
    b = rand(1, cols)
    y, buf = guarded(rows, cols, ty)
    spans = 1 if offsets is None else len(offsets) - 1
    mean, rstd = torch.empty(spans, groups, device="cuda"), torch.full((spans, groups), 7.0, device="cuda")
    dev = None if offsets is None else torch.tensor(offsets, device="cuda")
    xs.group_norm(executor, x, groups, None, b, 1e-5, y, offsets=dev, activation="relu", mean=mean, rstd=rstd)
    assert torch.isfinite(mean).all() and not rstd.any()
    inner = slice(0, rows) if offsets is None else slice(offsets[0], offsets[-1])
    assert torch.equal(y[inner], b.clamp(min=0).to(ty).expand(rows, cols)[inner])
