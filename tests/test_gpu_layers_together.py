"""GPU tests of the layer operators as they are used together: a training step of a norm over the graphs of a batch,
gated projections and their orthogonalised update, and the same layer served in 8 bits; calls from several threads at
once; a call on tensors that another device's context is not current for; long offsets.

The run's tolerance is that of its 16-bit roundings: an intermediate is off by U = 2^-11 (fp16) of itself, a sum of n
products of two rounded factors by 2 U sqrt(n) of its terms' root mean square sum where the roundings are independent;
the bounds below take 8 times that.
"""
import os
import subprocess
import sys
import threading

import pytest
import torch

import xspmm_b200 as xs
from xspmm_b200 import _lib

pytestmark = pytest.mark.gpu

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rand(seed, *shape, dtype=f32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def near(got, ref, rel):
    ref = ref.double()
    off = torch.linalg.vector_norm(got.double() - ref).item()
    assert off <= rel * torch.linalg.vector_norm(ref).item(), off / torch.linalg.vector_norm(ref).item()


def norm64(x, off, groups, w, b, eps):
    parts = []
    for lo, hi in zip(off[:-1], off[1:]):
        v = x[lo:hi].double().reshape(hi - lo, groups, x.shape[1] // groups)
        if hi > lo:
            m = v.mean((0, 2), keepdim=True)
            v = (v - m) / torch.sqrt(((v - m) ** 2).mean((0, 2), keepdim=True) + eps)
        parts.append(v.reshape(hi - lo, x.shape[1]))
    return torch.cat(parts) * w.double() + b.double()


@pytest.mark.parametrize("rows,cols,inner,groups", [(700, 128, 160, 8), (333, 90, 77, 9)])
def test_training_step(executor, rows, cols, inner, groups):
    """group norm with silu -> gated projections, back through both, and the weights' orthogonalised updates."""
    U = 2.0 ** -11
    off = [0, 100, 100, 101, rows]
    dev = torch.tensor(off, device="cuda")
    x, dy = rand(1, rows, cols), rand(2, rows, inner, dtype=f16)
    w, b = 1.0 + rand(3, cols, scale=0.2), rand(4, cols, scale=0.1)
    wg, wu = rand(5, inner, cols, dtype=f16, scale=cols ** -0.5), rand(6, inner, cols, dtype=f16, scale=cols ** -0.5)
    n, y = torch.empty(rows, cols, dtype=f16, device="cuda"), torch.empty(rows, inner, dtype=f16, device="cuda")
    gate, up, dn = torch.empty_like(y), torch.empty_like(y), torch.empty_like(n)
    mean, rstd = torch.empty(4, groups, device="cuda"), torch.empty(4, groups, device="cuda")
    dwg, dwu, dx = torch.empty_like(wg), torch.empty_like(wu), torch.empty_like(n)
    dw, db, step = torch.empty_like(w), torch.empty_like(b), torch.empty_like(wg)
    xs.group_norm(executor, x, groups, w, b, 1e-5, n, offsets=dev, activation="silu", mean=mean, rstd=rstd)
    xs.gated_ffn(executor, n, wg, wu, y, "silu", gate, up)
    xs.gated_ffn_backward(executor, dy, n, wg, wu, gate, up, dn, dwg, dwu)
    xs.group_norm_backward(executor, dn, x, groups, w, b, mean, rstd, dx, dw, db, offsets=dev, activation="silu")
    xs.orthogonalize(executor, dwg, step)

    leaves = [t.double().requires_grad_() for t in (x, w, b, wg, wu)]
    z = norm64(leaves[0], off, groups, leaves[1], leaves[2], 1e-5)
    h = torch.nn.functional.silu(z)
    out = torch.nn.functional.silu(h @ leaves[3].t()) * (h @ leaves[4].t())
    out.backward(dy.double())
    near(y, out.detach(), 8 * U)
    for got, leaf, deep in ((dwg, leaves[3], 2), (dwu, leaves[4], 2), (dx, leaves[0], 3), (dw, leaves[1], 3), (db, leaves[2], 3)):
        near(got, leaf.grad, 8 * deep * U)
    u, _, v = torch.linalg.svd(dwg.double(), full_matrices=False)  # the update's directions are the gradient's
    s = torch.diagonal(u.t() @ step.double() @ v.t())
    assert s.min().item() > 0 and s.max().item() < 1.21
    rest = u.t() @ step.double() @ v.t() - torch.diag(s)
    assert torch.linalg.vector_norm(rest).item() <= 8 * U * len(s) ** 0.5 * 2


@pytest.mark.parametrize("rows", [1, 12, 100, 400])
def test_served_in_8_bits(executor, rows):
    """group norm -> 8-bit rows -> product with an 8-bit weight: within the steps of both, 1 / 254 of a row's largest."""
    cols, inner = 256, 300
    x, w = rand(1, rows, cols, dtype=bf16), rand(2, inner, cols, dtype=bf16)
    wq, ws = torch.empty(inner, cols, dtype=torch.int8, device="cuda"), torch.empty(inner, device="cuda")
    xs.quantize_rows(executor, w, wq, ws)
    n = torch.empty_like(x)
    q, s = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    y = torch.empty(rows, inner, device="cuda")
    xs.group_norm(executor, x, 8, None, None, 1e-5, n, activation="gelu")
    xs.quantize_rows(executor, n, q, s)
    xs.linear_int8(executor, q, s, wq, ws, y)
    ref = n.double() @ w.double().t()
    # each factor is off by half a step at most
    ex, ew = s.double()[:, None] / 2, ws.double() / 2
    bound = ex * w.double().abs().sum(1) + ew * n.double().abs().sum(1, keepdim=True) + cols * ex * ew
    assert ((y.double() - ref).abs() <= bound * 1.001).all()


def test_the_example_with_orthogonal_updates():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "gated_graph_layer.py"), "--nodes-log2", "10", "--steps", "2",
                        "--update", "orthogonal"], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "loss" in r.stdout, r.stderr[-2000:]


def test_threads_with_their_own_executors(executor):
    """Calls of every operator from several threads at once, each with its executor, stream and tensors."""
    failures = []

    def work(seed):
        ex, stream = xs.CudaExecutor(0), torch.cuda.Stream()
        with torch.cuda.stream(stream):
            rows, cols = 300 + 37 * seed, 64 + 32 * seed
            x = rand(seed, rows, cols, dtype=f16)
            off = torch.tensor([0, 10, rows], device="cuda")

            def call():
                y, u = torch.empty_like(x), torch.empty_like(x)
                q, s = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
                p = torch.empty(rows, rows, dtype=f16, device="cuda")
                dw = torch.empty(cols, device="cuda")
                mean, rstd = torch.empty(2, 8, device="cuda"), torch.empty(2, 8, device="cuda")
                xs.group_norm(ex, x, 8, None, None, 1e-5, y, offsets=off, activation="silu", mean=mean, rstd=rstd)
                xs.group_norm_backward(ex, y, x, 8, None, None, mean, rstd, None, dw, offsets=off, activation="silu")
                xs.quantize_rows(ex, y, q, s)
                xs.linear_int8(ex, q, s, q, s, p)
                xs.orthogonalize(ex, x, u)
                return y, dw, q, s, p, u

            first = call()
            for _ in range(30):
                if not all(torch.equal(a, b) for a, b in zip(first, call())):
                    failures.append(seed)
                    break
            stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def test_offsets_past_32_bits(executor):
    """Element offsets above 2^31: the last rows of a matrix of 2^31 + elements."""
    cols = 4096
    rows = (1 << 31) // cols + 300
    x = torch.zeros(rows, cols, dtype=f16, device="cuda")
    tail = rand(1, 300, cols, dtype=f16)
    x[-300:] = tail
    y = torch.zeros_like(x)
    off = torch.tensor([rows - 300, rows], device="cuda")
    xs.group_norm(executor, x, 64, None, None, 1e-5, y, offsets=off, activation="relu")
    small = torch.empty_like(tail)
    xs.group_norm(executor, tail, 64, None, None, 1e-5, small, activation="relu")
    near(y[-300:], small, 2.0 ** -10)
    assert not y[:rows - 300].any()
    q, s = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    xs.quantize_rows(executor, x, q, s)
    q2, s2 = torch.empty(300, cols, dtype=torch.int8, device="cuda"), torch.empty(300, device="cuda")
    xs.quantize_rows(executor, tail, q2, s2)
    assert torch.equal(q[-300:], q2) and torch.equal(s[-300:], s2) and not s[:rows - 300].any()
    w, ws = q2[:64].contiguous(), s2[:64].contiguous()
    p, p2 = torch.empty(rows, 64, dtype=f16, device="cuda"), torch.empty(300, 64, dtype=f16, device="cuda")
    xs.linear_int8(executor, q, s, w, ws, p)
    xs.linear_int8(executor, q2, s2, w, ws, p2)
    assert torch.equal(p[-300:], p2) and not p[:rows - 300].any()


def _calls(ex):
    """A call of each operator through the C ABI with kernels of every kind, and its outputs; call() returns the statuses."""
    device, L, h = ex.device, _lib.lib(), ex.handle
    x = rand(1, 300, 160, dtype=f16).to(device)
    off = torch.tensor([0, 7, 300], device=device)
    y, dx, u = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    q, s = torch.zeros(300, 160, dtype=torch.int8, device=device), torch.zeros(300, device=device)
    p = torch.zeros(300, 300, dtype=f16, device=device)
    mean, rstd, dw = (torch.zeros(*n, device=device) for n in ((2, 8), (2, 8), (160,)))
    a = lambda t: t.data_ptr()  # noqa: E731
    torch.cuda.synchronize(device)

    def call():
        return [L.xspmm_group_norm_f16f16(h, 300, 160, 8, 2, a(off), a(x), 160, None, None, 1e-5, 0, a(y), 160, a(mean), a(rstd)),
                L.xspmm_group_norm_backward_f16f16(h, 300, 160, 8, 2, a(off), a(y), 160, a(x), 160, None, None, a(mean), a(rstd), 0,
                                                   a(dx), 160, a(dw), None),
                L.xspmm_quantize_rows_f16(h, 300, 160, a(y), 160, a(q), 160, a(s)),
                L.xspmm_linear_int8_f16(h, 300, 160, 300, a(q), 160, a(s), a(q), 160, a(s), None, a(p), 300),
                L.xspmm_orthogonalize_f16f16(h, 300, 160, a(x), 160, 5, 1e-7, a(u), 160)]

    return call, (y, dx, q, s, p, u, mean, rstd, dw, x, off)


def test_a_threads_first_cuda_calls(executor):
    """A host thread that has not touched the GPU has no device's context current; every operator runs from it."""
    call, here = _calls(executor)
    other, there = _calls(executor)
    assert call() == [0] * 5
    statuses = []
    thread = threading.Thread(target=lambda: statuses.extend(other()))
    thread.start()
    thread.join()
    assert statuses == [0] * 5, _lib.lib().xspmm_last_error()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(here, there))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device_than_the_current_one(executor):
    call, here = _calls(executor)
    assert torch.cuda.current_device() == 0
    other, there = _calls(xs.CudaExecutor(1))
    assert call() == [0] * 5 and other() == [0] * 5
    assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(0)
    torch.cuda.synchronize(1)
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(here, there))


def test_offsets_past_32_bits_in_the_gradient(executor):
    """The gradient of the last rows of matrices of 2^31 + elements; the rows before are in no sample and stay."""
    cols, tail = 4096, 300
    rows = (1 << 31) // cols + tail
    x, dy = (torch.zeros(rows, cols, dtype=f16, device="cuda") for _ in range(2))
    small = [rand(k, tail, cols, dtype=f16) for k in (1, 2)]
    x[-tail:], dy[-tail:] = small
    mean, rstd = rand(3, 1, 64, scale=0.1), rand(4, 1, 64).abs() + 0.5
    outs = []
    for xx, dd, off in ((x, dy, torch.tensor([rows - tail, rows], device="cuda")), (small[0], small[1], None)):
        dx, dw, db = torch.zeros_like(xx), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
        xs.group_norm_backward(executor, dd, xx, 64, None, None, mean, rstd, dx, dw, db, offsets=off, activation="silu")
        outs.append((dx, dw, db))
    (dx, dw, db), (sdx, sdw, sdb) = outs
    near(dx[-tail:], sdx, 2.0 ** -10)
    near(dw, sdw, 2.0 ** -18)
    near(db, sdb, 2.0 ** -18)
    assert not dx[:rows - tail].any()


def test_product_of_more_than_32_bits_of_elements(executor):
    """y of 2^31 + elements: its last rows are those of the product of the last rows alone."""
    K, F = 16, 66000
    rows = (1 << 31) // F + 500
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x, w = (torch.randint(-128, 128, (n, K), generator=g, device="cuda", dtype=torch.int8) for n in (rows, F))
    s, ws = rand(2, rows), rand(3, F)
    y, part = torch.empty(rows, F, dtype=f16, device="cuda"), torch.empty(400, F, dtype=f16, device="cuda")
    xs.linear_int8(executor, x, s, w, ws, y)
    xs.linear_int8(executor, x[-400:], s[-400:], w, ws, part)
    assert torch.equal(y[-400:], part)


def test_update_of_more_than_32_bits_of_elements(executor):
    """20 rows of 2^31 / 20 + columns: y = P g with a 20 x 20 matrix P, from g's products with itself."""
    m, n, slab = 20, (1 << 31) // 20 + 1000, 1 << 22
    g = torch.empty(m, n, dtype=f16, device="cuda")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    for c in range(0, n, slab):
        g[:, c:c + slab] = torch.randn(m, min(slab, n - c), generator=gen, device="cuda") * (1.0 + torch.arange(m, device="cuda"))[:, None]
    y = torch.zeros_like(g)
    xs.orthogonalize(executor, g, y)
    a = torch.zeros(m, m, dtype=torch.float64, device="cuda")
    for c in range(0, n, slab):
        v = g[:, c:c + slab].double()
        a += v @ v.t()
    norm = torch.sqrt(torch.diagonal(a).sum())
    a /= norm * norm
    p = torch.eye(m, dtype=torch.float64, device="cuda") / norm
    for _ in range(5):
        step = 3.4445 * torch.eye(m, dtype=torch.float64, device="cuda") - 4.7750 * a + 2.0315 * (a @ a)
        p, a = step @ p, step @ a @ step
    for c in (0, n // 2, n - 100_000):
        ref = p @ g[:, c:c + 100_000].double()
        near(y[:, c:c + 100_000], ref, 2.0 ** -11 + 2.0 ** -13)


def test_two_captured_graphs_at_once(executor):
    """Graphs of the same calls on different inputs, replayed side by side on two streams: each has its own scratch."""
    jobs = []
    for seed in (1, 2):
        x = rand(seed, 30000, 64, dtype=f16)
        g = rand(seed + 2, 400, 530, dtype=f16)
        off = torch.tensor([0, 7, 20000, 29990], device="cuda")
        y, dx, u = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(g)
        q, s = torch.empty(400, 530, dtype=torch.int8, device="cuda"), torch.empty(400, device="cuda")
        p = torch.empty(400, 400, dtype=f16, device="cuda")
        mean, rstd, dw = torch.zeros(3, 8, device="cuda"), torch.zeros(3, 8, device="cuda"), torch.zeros(64, device="cuda")

        def call(x=x, g=g, off=off, y=y, dx=dx, u=u, q=q, s=s, p=p, mean=mean, rstd=rstd, dw=dw):
            xs.group_norm(executor, x, 8, None, None, 1e-5, y, offsets=off, activation="silu", mean=mean, rstd=rstd)
            xs.group_norm_backward(executor, y, x, 8, None, None, mean, rstd, dx, dw, offsets=off, activation="silu")
            xs.quantize_rows(executor, g, q, s)
            xs.linear_int8(executor, q, s, q, s, p)
            xs.orthogonalize(executor, g, u)

        call()
        outs = (y, dx, u, q, s, p, mean, rstd, dw)
        want = [t.clone() for t in outs]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for t in outs:
            t.zero_()
        jobs.append((graph, torch.cuda.Stream(), outs, want, call))  # call keeps the inputs that the graph reads
    torch.cuda.synchronize()
    for _ in range(40):
        for graph, stream, _, _, _ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, outs, want, _ in jobs:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
