"""GPU tests of the group norm at the ends of its range: features of large magnitude, offsets that decrease,
sums of many terms."""
import math

import pytest
import torch

import test_gpu_group_norm
import xspmm_b200 as xs
from test_gpu_group_norm import U, bf16, check_backward, check_forward, f16, f32, guarded, outside_untouched, rand, value

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


# of 50000 rows: long samples that no or not every chunk finds, since a short or empty one hides them
DECREASING = [[0, 50000, 100, 200], [100, 200, 0, 50000], [0, 30000, 20000, 50000], [50000, 0, 50000], [0, 50000, 0, 50000],
              [0, 20000, 49000, 10000, 50000], [1 << 40, -5, 1 << 40, 7]]


@pytest.mark.parametrize("cols,groups", [(128, 32), (33, 3), (300, 1)])
@pytest.mark.parametrize("offsets", DECREASING)
def test_decreasing_offsets_take_nothing_from_earlier_calls(executor, offsets, cols, groups):
    """What is written is the same after calls that left different sums in the pool's memory, and nothing outside is."""
    rows = 50000
    x, dy = rand(1, rows, cols, dtype=bf16), rand(2, rows, cols, dtype=bf16)
    off, fine = torch.tensor(offsets, device="cuda"), torch.tensor([0] * (len(offsets) - 1) + [rows], device="cuda")
    samples = len(offsets) - 1
    got = []
    for scale in (1.0, 3.0):
        spare, dw, db = torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
        mean, rstd = torch.zeros(samples, groups, device="cuda"), torch.ones(samples, groups, device="cuda")
        torch.cuda.synchronize()
        xs.group_norm(executor, x * scale, groups, None, None, 1e-5, spare, offsets=fine, mean=mean, rstd=rstd)
        y, ybuf = guarded(rows, cols, bf16)
        mean, rstd = torch.full((samples, groups), 7.0, device="cuda"), torch.full((samples, groups), 7.0, device="cuda")
        xs.group_norm(executor, x, groups, None, None, 1e-5, y, offsets=off, activation="silu", mean=mean, rstd=rstd)
        one, zero = torch.ones(samples, groups, device="cuda"), torch.zeros(samples, groups, device="cuda")
        xs.group_norm_backward(executor, dy * scale, x, groups, None, None, zero, one, spare, dw, db, offsets=fine)
        dx, dbuf = guarded(rows, cols, bf16)
        dw, db = torch.full((cols,), 7.0, device="cuda"), torch.full((cols,), 7.0, device="cuda")
        xs.group_norm_backward(executor, dy, x, groups, None, None, zero, one, dx, dw, db, offsets=off)
        outside_untouched(y, ybuf)
        outside_untouched(dx, dbuf)
        got.append((y, mean, rstd, dx, dw, db))
    for a, b in zip(*got):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def test_a_sample_that_a_later_one_hides_has_no_statistics(executor):
    x = rand(1, 50000, 128, dtype=f16)
    y, mean = torch.zeros_like(x), torch.zeros(3, 32, device="cuda")
    xs.group_norm(executor, x, 32, None, None, 1e-5, y, offsets=torch.tensor([0, 50000, 100, 200], device="cuda"), mean=mean)
    assert mean[0].isnan().all() and not mean[1].any() and mean[2].isfinite().all()


@pytest.mark.parametrize("rows,cols,samples", [(1 << 24, 128, 1), (1 << 26, 8, 1 << 26)])
def test_sums_of_equal_terms(executor, rows, cols, samples):
    """dy = 1 + 2^-13 - 2^-20 and xh = 1 everywhere: added up one after the other, every term past the 2048th loses its
    fraction, 7000 in a row 8.6e-5 of the sum. 1024 + 32 roundings of half a step are 6.3e-5."""
    term = 1.0 + 2.0 ** -13 - 2.0 ** -20
    x, dy = torch.ones(rows, cols, device="cuda"), torch.full((rows, cols), term, device="cuda")
    mean, rstd = torch.zeros(samples, 1, device="cuda"), torch.ones(samples, 1, device="cuda")
    off = None if samples == 1 else torch.arange(samples + 1, device="cuda")
    dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    xs.group_norm_backward(executor, dy, x, 1, None, None, mean, rstd, None, dw, db, offsets=off)
    want = rows * term
    for got in (dw, db):
        assert (got.double() - want).abs().max().item() <= 1.01 * (1024 + 32) * 2.0 ** -24 * want


class EqualLengths(test_gpu_group_norm.Ref):
    """The 64-bit sums of samples of one length, all at once."""

    def mean_of(self, v):
        return v.reshape(len(self.spans), -1, self.groups, self.width).sum((1, 3)) * self.per

    def spread(self, v, rows):
        v = v.expand(len(self.spans), self.groups).repeat_interleave(self.width, 1)
        return v.repeat_interleave(rows // len(self.spans), 0)


@pytest.mark.parametrize("tx,ty", [(f16, f16), (f32, f32), (f32, bf16)])
@pytest.mark.parametrize("samples,length,cols,groups", [(40000, 3, 64, 8), (40000, 2, 21, 3), (3000, 40, 640, 5), (6000, 1, 300, 1)])
def test_walks_over_many_samples(executor, monkeypatch, samples, length, cols, groups, tx, ty):
    """So many samples that every warp, or CTA, of the gradient takes several in turn."""
    monkeypatch.setattr(test_gpu_group_norm, "Ref", EqualLengths)
    rows = samples * length
    offsets = list(range(0, rows + 1, length))
    x, dy = rand(21, rows, cols, dtype=tx, shift=0.5), rand(22, rows, cols, dtype=ty, shift=0.5)
    w, b = rand(23, cols, scale=0.2, shift=1.0), rand(24, cols, scale=0.1)
    y, ybuf = guarded(rows, cols, ty)
    check_forward(executor, x, groups, w, b, 1e-5, y, offsets, "silu", ybuf)
    dx, dbuf = guarded(rows, cols, ty)
    check_backward(executor, dy, x, groups, w, b, offsets, "silu", dx, dbuf)
