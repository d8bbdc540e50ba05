"""GPU tests of the group norm with an activation, forward and backward, against plain restatements in 64 bits.

Tolerances, element by element. U[T] is the largest relative error of one rounding to type T, TINY[T] the
largest absolute one among its subnormals. No sum adds more than 1024 terms one after the other (longer ones are
joined from partial sums), so a sum of n fp32 terms is within H(n) = (min(n, 1024) + 32) * 2^-24 of the sum of
their magnitudes. E = 2^-20 covers the roundings and the exponential of an elementwise formula. An error e of z
moves the activation by at most 1.13 e and its slope by at most 1.2 e (the largest first and second derivatives
of gelu, the steepest of them).
"""
import math

import pytest
import torch

import xspmm_b200 as xs

pytestmark = pytest.mark.gpu

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32
U = {f16: 2.0 ** -11, bf16: 2.0 ** -8, f32: 2.0 ** -24}
TINY = {f16: 2.0 ** -25, bf16: 2.0 ** -134, f32: 2.0 ** -150}
E = 2.0 ** -20
TYPES = [(f16, f16), (bf16, bf16), (f32, f32), (f32, f16), (f32, bf16)]
ACTS = [None, "silu", "gelu", "relu", "sigmoid"]


def H(n):
    return (torch.clamp(n, max=1024.0) + 32.0) * 2.0 ** -24


def rand(seed, *shape, dtype=f32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def close(got, ref, err, what=""):
    T = got.dtype
    tol = 1.01 * (err + U[T] * ref.abs()) + TINY[T]
    assert torch.isfinite(got).all(), what
    off = (got.double() - ref).abs()
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: off by {off.max().item():.3e}, over the bound by {worst:.3e}"


def guarded(rows, cols, dtype, ld=None, fill=7.0):
    ld = ld or cols
    buf = torch.full((rows * ld + 64,), fill, dtype=dtype, device="cuda")
    return buf.as_strided((rows, cols), (ld, 1)), buf


def outside_untouched(view, buf, fill=7.0):
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep.as_strided(view.shape, view.stride()).fill_(False)
    assert bool((buf[keep] == fill).all()), "written outside the output"


def value(name, z):
    if name is None:
        return z
    if name == "silu":
        return z * torch.special.expit(z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return z.clamp(min=0) if name == "relu" else torch.special.expit(z)


def slope(name, z):
    if name is None:
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.special.expit(z)
    return s * (1 + z * torch.special.expit(-z)) if name == "silu" else s * torch.special.expit(-z)


class Ref:
    """Samples' sums in 64 bits, one sample after the other."""

    def __init__(self, offsets, rows, cols, groups):
        self.spans = [(0, rows)] if offsets is None else list(zip(offsets[:-1], offsets[1:]))
        self.groups, self.cols, self.width = groups, cols, cols // groups
        self.first, self.last = self.spans[0][0], self.spans[-1][1]
        self.n = torch.tensor([max(b - a, 0) * self.width for a, b in self.spans], dtype=torch.float64, device="cuda")[:, None]
        self.per = 1.0 / self.n.clamp(min=1.0)

    def mean_of(self, v):  # over each sample's rows and group's columns: samples x groups
        v = v.reshape(v.shape[0], self.groups, self.width).sum(2)
        return torch.stack([v[a:b].sum(0) for a, b in self.spans]) * self.per

    def spread(self, v, rows):  # samples x groups (or x 1) to rows x cols; 0 outside the samples
        out = torch.zeros(rows, self.cols, dtype=torch.float64, device="cuda")
        v = v.expand(len(self.spans), self.groups).repeat_interleave(self.width, 1)
        for i, (a, b) in enumerate(self.spans):
            out[a:b] = v[i]
        return out

    def statistics(self, x, eps):
        rows = x.shape[0]
        x = x.double()
        mean = self.mean_of(x)
        d = x - self.spread(mean, rows)
        return mean, 1.0 / torch.sqrt(self.mean_of(d * d) + eps)


def check_forward(ex, x, groups, w, b, eps, y, offsets, act, ybuf=None):
    rows, cols = x.shape
    ref = Ref(offsets, rows, cols, groups)
    samples = len(ref.spans)
    mean, rstd = torch.empty(samples, groups, device="cuda"), torch.empty(samples, groups, device="cuda")
    before = y.clone()
    dev = None if offsets is None else torch.tensor(offsets, device="cuda")
    x64 = x.double()
    xs.group_norm(ex, x, groups, w, b, eps, y, offsets=dev, activation=act, mean=mean, rstd=rstd)
    rm, rr = ref.statistics(x64, eps)
    em = H(ref.n) * ref.mean_of(x64.abs()) + E * rm.abs()
    d = x64 - ref.spread(rm, rows)
    er = rr * (H(ref.n) + 0.5 * (em * rr) ** 2 + 2.0 ** -22)
    close(mean, rm, em, "mean")
    close(rstd, rr, er, "rstd")
    s = lambda v: ref.spread(v, rows)  # noqa: E731
    wd, bd = (torch.ones(cols, device="cuda") if w is None else w).double(), (torch.zeros(cols, device="cuda") if b is None else b).double()
    xh = d * s(rr)
    z = xh * wd + bd
    ez = wd.abs() * (s(em * rr) + xh.abs() * (s(er / rr) + E)) + E * (z.abs() + bd.abs())
    inner = slice(ref.first, ref.last)
    want = value(act, z)
    close(y[inner], want[inner], (1.13 * ez + 4 * E * want.abs())[inner], f"y ({act})")
    for part in (slice(0, ref.first), slice(ref.last, rows)):
        assert torch.equal(y[part], before[part]), "rows outside the samples changed"
    if ybuf is not None:
        outside_untouched(y, ybuf)
    return mean, rstd


def check_backward(ex, dy, x, groups, w, b, offsets, act, dx, xbuf=None, eps=1e-5):
    rows, cols = x.shape
    ref = Ref(offsets, rows, cols, groups)
    rm, rr = ref.statistics(x, eps)
    mean, rstd = rm.float(), rr.float()
    dw, db = torch.full((cols,), 3.0, device="cuda"), torch.full((cols,), 3.0, device="cuda")
    before = dx.clone()
    dev = None if offsets is None else torch.tensor(offsets, device="cuda")
    g = dy.double()
    s = lambda v: ref.spread(v, rows)  # noqa: E731
    inside = s(torch.ones_like(rr)) > 0
    wd, bd = (torch.ones(cols, device="cuda") if w is None else w).double(), (torch.zeros(cols, device="cuda") if b is None else b).double()
    m, r = s(mean.double()), s(rstd.double())
    xh = (x.double() - m) * r
    z = xh * wd + bd
    if act == "relu":  # the sign is that of the fp32 operations, one after the other
        z = (((x.float() - m.float()) * r.float()) * wd.float() + bd.float()).double()
    dz = torch.where(inside, g * slope(act, z), torch.zeros_like(g))
    xh = torch.where(inside, xh, torch.zeros_like(xh))
    xs.group_norm_backward(ex, dy, x, groups, w, b, mean, rstd, dx, dw, db, offsets=dev, activation=act)
    t = dz * wd
    # xh: two roundings; z: two more
    exh = 2.0 ** -23 * xh.abs()
    ez = 2.0 ** -22 * ((xh * wd).abs() + bd.abs())
    edz = g.abs() * ((0.0 if act in (None, "relu") else 1.0) * (1.2 * ez + 4 * E * (1.0 + z.abs()) * slope(act, z).abs())) + E * dz.abs()
    et = wd.abs() * edz + E * t.abs()
    c1, c2 = ref.mean_of(t), ref.mean_of(t * xh)
    h = H(ref.n) + E
    e1 = h * ref.mean_of(t.abs()) + ref.mean_of(et)
    e2 = h * ref.mean_of((t * xh).abs()) + ref.mean_of(et * xh.abs() + t.abs() * exh)
    dxr = r * (t - s(c1) - xh * s(c2))
    err = r * (et + s(e1) + xh.abs() * s(e2) + exh * s(c2).abs() + E * (t.abs() + s(c1).abs() + (xh * s(c2)).abs()))
    inner = slice(ref.first, ref.last)
    close(dx[inner], dxr[inner], err[inner], f"dx ({act})")
    total = torch.tensor(float(ref.last - ref.first), dtype=torch.float64, device="cuda")
    hr = H(total) + E
    close(dw, (dz * xh).sum(0), hr * (dz * xh).abs().sum(0) + (edz * xh.abs() + dz.abs() * exh).sum(0), "dweight")
    close(db, dz.sum(0), hr * dz.abs().sum(0) + edz.sum(0), "dbias")
    for part in (slice(0, ref.first), slice(ref.last, rows)):
        assert torch.equal(dx[part], before[part]), "rows outside the samples changed"
    if xbuf is not None:
        outside_untouched(dx, xbuf)
    return dw, db, mean, rstd


# rows, cols, groups, offsets
CASES = [
    (1, 1, 1, None), (1, 64, 4, None), (5, 7, 7, None), (3, 21, 3, [0, 1, 3]), (64, 32, 1, None),
    (301, 84, 12, None), (200, 129, 43, [0, 64, 64, 65, 200]), (1000, 128, 32, [0, 1000]),
    (999, 256, 32, [3, 10, 10, 400, 990]), (40, 1021, 1, [0, 13, 40]), (33, 2050, 2, None), (7, 6000, 4, [0, 3, 7]),
    (3, 16384, 1, None), (2, 20480, 5, [0, 1, 2]), (5000, 24, 3, None), (2049, 40, 5, [0, 2049]),
    (20000, 16, 16, [0, 5, 19000, 19001, 20000]), (513, 96, 2, list(range(0, 514))), (4100, 65, 13, [100, 4000, 4050]),
]


def data(i, tx, ty):
    rows, cols, groups, offsets = CASES[i]
    x = rand(i, rows, cols, dtype=tx, scale=1.5, shift=0.25)
    return x, rand(i + 100, rows, cols, dtype=ty), groups, rand(1, cols, scale=0.2, shift=1.0), rand(2, cols, scale=0.1), offsets


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("i", range(len(CASES)))
def test_forward(executor, i, tx, ty):
    x, _, groups, w, b, offsets = data(i, tx, ty)
    y, buf = guarded(*x.shape, ty)
    check_forward(executor, x, groups, w, b, 1e-5, y, offsets, ACTS[i % 5], buf)


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("i", range(len(CASES)))
def test_backward(executor, i, tx, ty):
    x, dy, groups, w, b, offsets = data(i, tx, ty)
    dx, buf = guarded(*x.shape, ty)
    dw, db, mean, rstd = check_backward(executor, dy, x, groups, w, b, offsets, ACTS[i % 5], dx, buf)
    # the parts alone are the same numbers
    dev = None if offsets is None else torch.tensor(offsets, device="cuda")
    kw = dict(offsets=dev, activation=ACTS[i % 5])
    dx2, dw2, db2 = torch.full_like(dx, 7.0), torch.empty_like(dw), torch.empty_like(db)
    xs.group_norm_backward(executor, dy, x, groups, w, b, mean, rstd, dx2, **kw)
    xs.group_norm_backward(executor, dy, x, groups, w, b, mean, rstd, None, dw2, None, **kw)
    xs.group_norm_backward(executor, dy, x, groups, w, b, mean, rstd, None, None, db2, **kw)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and torch.equal(db, db2)


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations(executor, tx, ty, act):
    """Every activation with every type, gates from -40 to 40 among them, on aligned and odd widths."""
    for cols, groups in ((64, 8), (63, 9)):
        x = rand(5, 70, cols, dtype=tx, scale=2.0, shift=-0.5)
        w, b = rand(6, cols, scale=3.0), rand(7, cols, scale=6.0)
        w[3], b[5], b[6] = 12.0, 40.0, -40.0
        check_forward(executor, x, groups, w, b, 1e-5, torch.zeros(70, cols, dtype=ty, device="cuda"), [0, 20, 70], act)
        check_backward(executor, rand(8, 70, cols, dtype=ty), x, groups, w, b, [0, 20, 70], act,
                       torch.zeros(70, cols, dtype=ty, device="cuda"))


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("pad", [1, 8])
def test_row_strides_and_unaligned_starts(executor, tx, ty, pad):
    rows, cols = 260, 96
    offsets = [0, 100, 103, 260]
    x = rand(9, rows, cols + 2 * pad, dtype=tx)[:, pad:pad + cols]
    dy = rand(10, rows, cols + pad, dtype=ty)[:, :cols]
    y, ybuf = guarded(rows, cols, ty, ld=cols + pad)
    check_forward(executor, x, 12, rand(1, cols), rand(2, cols), 1e-5, y, offsets, "silu", ybuf)
    dx, dbuf = guarded(rows, cols, ty, ld=cols + 2 * pad)
    check_backward(executor, dy, x, 12, rand(1, cols), rand(2, cols), offsets, "silu", dx, dbuf)


def test_without_parameters_and_in_place(executor):
    x, dy = rand(3, 50, 96, dtype=bf16), rand(4, 50, 96, dtype=bf16)
    check_forward(executor, x.clone(), 6, None, None, 1e-5, torch.zeros_like(x), None, "gelu")
    one, zero = torch.ones(96, device="cuda"), torch.zeros(96, device="cuda")
    y1, y2 = torch.empty_like(x), x.clone()
    mean, rstd = torch.empty(1, 6, device="cuda"), torch.empty(1, 6, device="cuda")
    xs.group_norm(executor, x, 6, one, zero, 1e-5, y1, activation="silu", mean=mean, rstd=rstd)
    xs.group_norm(executor, y2, 6, None, None, 1e-5, y2, activation="silu")
    assert torch.equal(y1, y2)
    d1 = torch.empty_like(x)
    xs.group_norm_backward(executor, dy, x, 6, one, zero, mean, rstd, d1, activation="silu")
    xs.group_norm_backward(executor, dy, x, 6, None, None, mean, rstd, dy, activation="silu")
    assert torch.equal(d1, dy)


def test_nothing_to_do(executor):
    """No samples, no rows, empty samples only: weights' gradients are zero, statistics those of no values."""
    w = torch.ones(8, device="cuda")
    none = torch.empty(0, 8, device="cuda")
    m1 = torch.full((1, 2), 5.0, device="cuda")
    r1 = m1.clone()
    xs.group_norm(executor, none, 2, w, w, 0.25, none, mean=m1, rstd=r1)
    assert (m1 == 0).all() and (r1 == 2.0).all()
    dw, db = w.clone(), w.clone()
    xs.group_norm_backward(executor, none, none, 2, w, w, m1, r1, none, dw, db)
    assert not dw.any() and not db.any()
    x, y = rand(1, 6, 8), torch.full((6, 8), 7.0, device="cuda")
    for offsets in ([3], [2, 2, 2]):
        off = torch.tensor(offsets, device="cuda")
        m, r = torch.full((len(offsets) - 1, 2), 5.0, device="cuda"), torch.full((len(offsets) - 1, 2), 5.0, device="cuda")
        xs.group_norm(executor, x, 2, w, w, 0.25, y, offsets=off, mean=m, rstd=r)
        assert (y == 7.0).all() and (m == 0).all() and (r == 2.0).all()
        dw, db = w.clone(), w.clone()
        xs.group_norm_backward(executor, x, x, 2, w, w, m, r, y, dw, db, offsets=off)
        assert (y == 7.0).all() and not dw.any() and not db.any()


def test_constant_groups_large_means_and_outliers(executor):
    """A constant group has variance 0; a mean of 1e4 times the deviation and a row far off the others, first
    or not, keep the statistics' accuracy."""
    x = rand(11, 3000, 32, dtype=f32)
    x[:, :4] = 3.0
    x[:, 4:8] += 1e4
    x[0, 8:12] = 1e5
    x[1777, 12:16] = -1e6
    y = torch.zeros_like(x)
    mean, rstd = check_forward(executor, x, 8, None, None, 1e-5, y, None, None)
    assert mean[0, 0].item() == 3.0 and (y[:, :4] == 0).all()


def test_not_a_number_stays_in_its_sample_and_group(executor):
    x = rand(12, 90, 24, dtype=f16)
    x[40, 9], x[70, 20] = float("nan"), float("inf")
    y = torch.empty_like(x)
    xs.group_norm(executor, x, 3, None, None, 1e-5, y, offsets=torch.tensor([0, 30, 60, 90], device="cuda"),
                  activation="silu")
    bad = torch.zeros(90, 24, dtype=torch.bool, device="cuda")
    bad[30:60, 8:16] = True
    bad[60:90, 16:24] = True
    assert torch.isnan(y[30:60, 8:16]).all() and torch.isnan(y[60:90, 16:24]).any()
    assert torch.isfinite(y[~bad]).all()


def test_offsets_out_of_order_or_range_touch_nothing_outside(executor):
    x = rand(13, 50, 16, dtype=bf16)
    for offsets in ([0, 30, 20, 50], [-5, 10, 1 << 40], [60, 70], [50, 0], [1 << 62, -(1 << 62), 3]):
        off = torch.tensor(offsets, device="cuda")
        y, buf = guarded(50, 16, bf16)
        mean, rstd = torch.zeros(len(offsets) - 1, 4, device="cuda"), torch.ones(len(offsets) - 1, 4, device="cuda")
        xs.group_norm(executor, x, 4, None, None, 1e-5, y, offsets=off, activation="relu")
        dw, db = torch.empty(16, device="cuda"), torch.empty(16, device="cuda")
        xs.group_norm_backward(executor, x, x, 4, None, None, mean, rstd, y, dw, db, offsets=off)
        outside_untouched(y, buf)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_against_differences(executor, act):
    """The directional derivative of sum(dy * y), by central differences of the 64-bit formula."""
    rows, cols, groups, offsets, h = 23, 30, 5, [0, 9, 23], 1e-4
    x, w, b = rand(1, rows, cols), rand(2, cols, shift=1.0, scale=0.3), rand(3, cols)
    dy = rand(4, rows, cols)
    dirs = [rand(5 + k, *t.shape).double() for k, t in enumerate((x, w, b))]
    ref = Ref(offsets, rows, cols, groups)

    def loss(e):
        xe, we, be = (t.double() + e * d for t, d in zip((x, w, b), dirs))
        m, r = ref.statistics(xe, 1e-5)
        return (dy.double() * value(act, (xe - ref.spread(m, rows)) * ref.spread(r, rows) * we + be)).sum().item()

    m, r = ref.statistics(x, 1e-5)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    xs.group_norm_backward(executor, dy, x, groups, w, b, m.float(), r.float(), dx, dw, db,
                           offsets=torch.tensor(offsets, device="cuda"), activation=act)
    got = sum((g.double() * d).sum().item() for g, d in zip((dx, dw, db), dirs))
    want = (loss(h) - loss(-h)) / (2 * h)
    size = sum((g.double() * d).abs().sum().item() for g, d in zip((dx, dw, db), dirs))
    assert abs(got - want) <= 1e-5 * size


def test_streams_graphs_and_repeats(executor):
    """The same call on another stream, captured and replayed on new inputs, and repeated: the same numbers."""
    rows, cols, groups = 30000, 64, 8
    off = torch.tensor([0, 7, 20000, 29990], device="cuda")
    x, dy = rand(1, rows, cols, dtype=f16), rand(2, rows, cols, dtype=f16)
    w, b = rand(3, cols), rand(4, cols)

    def outputs():
        return (torch.zeros_like(x), torch.zeros(3, groups, device="cuda"), torch.zeros(3, groups, device="cuda"),
                torch.zeros_like(x), torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda"))

    def call(out):
        y, m, r, dx, dw, db = out
        xs.group_norm(executor, x, groups, w, b, 1e-5, y, offsets=off, activation="silu", mean=m, rstd=r)
        xs.group_norm_backward(executor, dy, x, groups, w, b, m, r, dx, dw, db, offsets=off, activation="silu")

    first, other, replayed = outputs(), outputs(), outputs()
    call(first)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(other)
    side.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    spare = outputs()
    with torch.cuda.graph(graph):
        call(replayed)
    with torch.cuda.graph(second):
        call(spare)
    x.mul_(-1.0)
    graph.replay()
    second.replay()
    torch.cuda.synchronize()
    again = outputs()
    call(again)
    torch.cuda.synchronize()
    for a, o in zip(first, other):
        assert torch.equal(a, o)
    for a, o, p in zip(again, replayed, spare):
        assert torch.equal(a, o) and torch.equal(a, p)


def mixed(cols, size):
    """Offsets of 3000 samples: mostly a few rows, some empty, one of more than a warp takes, one of more than a CTA."""
    lengths = [(7 * i) % 11 for i in range(3000)]
    lengths[100], lengths[1234], lengths[2990] = 70_000 // (cols * size) + 50, 400_000 // (cols * size) + 300, 40
    ends = torch.tensor([3] + lengths).cumsum(0).tolist()
    return ends, ends[-1] + 5


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("cols,groups", [(64, 8), (33, 11), (30, 1), (264, 2), (520, 1)])
def test_many_samples(executor, cols, groups, tx, ty):
    """Short samples by a warp each, middle ones by a CTA, long ones by all, side by side."""
    offsets, rows = mixed(cols, 2)
    x, dy = rand(21, rows, cols, dtype=tx, shift=0.5), rand(22, rows, cols, dtype=ty)
    w, b = rand(23, cols, scale=0.2, shift=1.0), rand(24, cols, scale=0.1)
    y, ybuf = guarded(rows, cols, ty)
    check_forward(executor, x, groups, w, b, 1e-5, y, offsets, "silu", ybuf)
    dx, dbuf = guarded(rows, cols, ty)
    check_backward(executor, dy, x, groups, w, b, offsets, "silu", dx, dbuf)


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("rows,cols,groups,offsets", [
    (30000, 128, 32, None), (30000, 33, 3, [0, 9000, 9000, 9001, 21000, 29999]), (9000, 640, 1, [5, 4000, 8990]),
    (40000, 8, 2, [1, 20000, 20001, 40000])])
def test_long_samples(executor, rows, cols, groups, offsets, tx, ty):
    """Samples cut into chunks, which begin and end inside them."""
    x, dy = rand(31, rows, cols, dtype=tx, shift=0.5), rand(32, rows, cols, dtype=ty)
    w, b = rand(33, cols, scale=0.2, shift=1.0), rand(34, cols, scale=0.1)
    y, ybuf = guarded(rows, cols, ty)
    check_forward(executor, x, groups, w, b, 1e-5, y, offsets, "gelu", ybuf)
    dx, dbuf = guarded(rows, cols, ty)
    check_backward(executor, dy, x, groups, w, b, offsets, "gelu", dx, dbuf)


@pytest.mark.parametrize("cols,groups", [(32, 4), (474, 2), (21, 3)])
def test_relu_slope_is_that_of_z_rounded_step_by_step(executor, cols, groups):
    """z is 0 where the rounded product is exactly -bias, and its slope is 0 there: dbias counts the rows with z > 0."""
    rows = 3000
    x, b = rand(41, rows, cols), rand(42, cols, scale=0.1)
    w = 1.0 + rand(43, cols, scale=0.2)
    mean, rstd = rand(44, 1, groups, scale=0.1), rand(45, 1, groups).abs() + 0.5
    width = cols // groups
    m, r = mean[0].repeat_interleave(width), rstd[0].repeat_interleave(width)
    rounded = ((x - m) * r) * w  # separate kernels: each operation rounded
    b = -rounded[torch.arange(cols, device="cuda") % rows, torch.arange(cols, device="cuda")]  # a zero in every column
    z = rounded + b
    assert int((z == 0).sum()) >= cols
    db = torch.empty(cols, device="cuda")
    xs.group_norm_backward(executor, torch.ones_like(x), x, groups, w, b, mean, rstd, None, None, db, activation="relu")
    assert torch.equal(db.long(), (z > 0).sum(0))


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("cols", [16, 23])
def test_gradient_of_groups_of_one_value_is_zero(executor, cols, tx, ty):
    """One row and one channel a group: y does not depend on x, and rstd (316 for eps 1e-5) multiplies no rounding."""
    rows = 40
    off = torch.arange(rows + 1, device="cuda")
    x, dy = rand(51, rows, cols, dtype=tx), rand(52, rows, cols, dtype=ty)
    w, b = rand(53, cols, shift=1.0, scale=0.2), rand(54, cols, scale=0.1)
    mean, rstd = torch.empty(rows, cols, device="cuda"), torch.empty(rows, cols, device="cuda")
    y, dx = torch.empty(rows, cols, dtype=ty, device="cuda"), torch.empty(rows, cols, dtype=ty, device="cuda")
    xs.group_norm(executor, x, cols, w, b, 1e-5, y, offsets=off, activation="silu", mean=mean, rstd=rstd)
    assert torch.equal(mean, x.float())
    xs.group_norm_backward(executor, dy, x, cols, w, b, mean, rstd, dx, offsets=off, activation="silu")
    assert not dx.any()
