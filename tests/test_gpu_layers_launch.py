"""GPU tests of the layer operators' launches: shared memory at the edges of what a launch may take unasked,
launches of one kernel from several threads, and a thread whose first CUDA call is one of them."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import xspmm_b200 as xs
from xspmm_b200 import _lib

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# Widths whose ring needs a little less than 48 KB, each instance's narrowest first: a wider row before
# it would have raised the kernel's limit for the process.
_WIDTHS = r"""
import torch
import xspmm_b200 as xs

ex = xs.CudaExecutor(0)
f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32


def run(D, tx, ty):
    g = torch.Generator(device="cuda")
    g.manual_seed(D)
    x = torch.randn(3, D, generator=g, device="cuda").to(tx)
    y, mean, rstd = torch.empty(3, D, dtype=ty, device="cuda"), torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    return x, y, mean, rstd


def same(got, ref):  # every rounding and sum of these widths stays far below this
    assert (got.double() - ref).abs().max().item() <= 2.0 ** -7 * ref.abs().max().item()


for tx, ty, widths in ((f16, f16, (12192, 12200, 12240, 12272)), (bf16, bf16, (12200, 12264)),
                       (f32, f32, (6096, 6100, 6120, 6136)), (f32, f16, (6100, 6132)), (f32, bf16, (6104, 6136))):
    for D in widths:
        x, y, mean, rstd = run(D, tx, ty)
        xs.layer_norm(ex, x, None, None, 1e-5, y, mean, rstd)
        d = x.double() - x.double().mean(1, keepdim=True)
        same(y, d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5))
for tx, ty, widths in ((f16, f16, (6056, 6064, 6080, 6112, 6128)), (bf16, bf16, (6080,)),
                       (f32, f32, (3028, 3036, 3040, 3064)), (f32, f16, (4032, 4040, 4064, 4080)), (f32, bf16, (4080,))):
    for D in widths:
        x, dx, mean, rstd = run(D, tx, ty)
        dy = x.flip(0).to(ty).contiguous()
        mean.fill_(0.25)
        rstd.fill_(0.5)
        dw, db = torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
        xs.layer_norm_backward(ex, dy, x, None, mean, rstd, dx, dw, db)
        xh, t = (x.double() - 0.25) * 0.5, dy.double()
        same(dx, 0.5 * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True)))
        same(dw, (t * xh).sum(0))
        same(db, t.sum(0))
print("done")
"""


def test_rings_of_a_little_less_than_48_kb(executor):
    r = subprocess.run([sys.executable, "-c", _WIDTHS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


def _gated(handle, rows, K, F):
    x, wg, wu = (torch.ones(r, K, dtype=torch.bfloat16, device="cuda") for r in (rows, F, F))
    y = torch.empty(rows, F, dtype=torch.bfloat16, device="cuda")
    args = (handle, rows, K, F, 2, x.data_ptr(), K, wg.data_ptr(), K, wu.data_ptr(), K, y.data_ptr(), F, None, None)
    return _lib.lib().xspmm_gated_ffn_bf16, args, y, float(K * K), (x, wg, wu)


def _norm(handle, cols):
    x, bias = torch.ones(2, cols, device="cuda"), torch.full((cols,), 0.75, device="cuda")
    y = torch.empty_like(x)
    args = (handle, 2, cols, x.data_ptr(), cols, None, bias.data_ptr(), 1e-5, y.data_ptr(), cols, None, None)
    return _lib.lib().xspmm_layer_norm_f32f32, args, y, 0.75, (x, bias)


# shapes of one kernel instance whose shared memory differs
@pytest.mark.parametrize("shapes", [[(_gated, 300, 32, 16), (_gated, 20000, 64, 256)],
                                    [(_gated, 100, 32, 8), (_gated, 100, 64, 20000)],
                                    [(_norm, 6300), (_norm, 8192)]])
def test_threads_with_their_own_executors(executor, shapes):
    """Each thread has its handle, stream and tensors; every call has to launch whatever size the others use.
    The entries are called without the Python checks between them, so that calls overlap."""
    failures = []
    start = threading.Barrier(2 * len(shapes))

    def work(make, *size):
        ex, stream = xs.CudaExecutor(0), torch.cuda.Stream()
        with torch.cuda.stream(stream):
            call, args, y, want, _inputs = make(ex.handle, *size)
            torch.cuda.current_stream().synchronize()
            start.wait(timeout=60)
            for _ in range(8000):
                if call(*args):
                    failures.append((make.__name__, size, _lib.lib().xspmm_last_error()))
                    break
            stream.synchronize()
            if not bool((y == want).all()):
                failures.append((make.__name__, size, "wrong result"))

    threads = [threading.Thread(target=work, args=s) for s in shapes for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


def test_a_threads_first_cuda_call(executor):
    """A host thread that has not touched the GPU yet has no context of its own to encode tensor maps in."""
    call, args, y, want, _inputs = _gated(executor.handle, 300, 32, 64)
    torch.cuda.synchronize()
    results = []
    thread = threading.Thread(target=lambda: results.append((call(*args), _lib.lib().xspmm_last_error())))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert results[0][0] == 0, results
    assert bool((y == want).all())
