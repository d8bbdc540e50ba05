"""GPU tests of the layer operators' launches: shared memory at the edges of what a launch may take unasked."""
import os
import subprocess
import sys

import pytest

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
